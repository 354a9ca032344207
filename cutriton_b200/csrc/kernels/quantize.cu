// QuantizeRows: FP16 rows to 8-bit integers with one scale a row.
//
//   s[m] = fl32(max_k |x[m, k]| / 127),  q[m, k] = round_half_even(x[m, k] / s[m])
//
// exactly, i.e. as if the quotient were not rounded before it is rounded to
// an integer. A row of zeros has s = 0 and q = 0. A row that holds an infinity
// or a NaN has s = inf or NaN and q = 0, so that a product with it is NaN.
//
// One pass over HBM (3 bytes an element). A warp (two to sixteen for long or
// few rows) takes whole rows and waits for no other one: each lane copies its
// vectors of 8 elements into a queue of its own in shared memory (cp.async),
// 9 KB a warp, finds the row's maximum, and reads them back to write the
// integers. So 216 KB of an SM's rows are under way while 24 warps compute,
// which takes 14 of the 16.7 lane instructions an element that full HBM rate
// leaves: the rounding, exact by comparing two, is half of them.
// 16384x8192: 67 us, 6.0 TB/s (with 16 warps 9 %, with 12 13 % more); with rows in
// registers, by blocks of 256 threads with two barriers a row, 96 us (and
// 16384x2048 52 us for 23).
//
// Element i of x and of q have the same flat index, so a vector of 8 elements
// that starts at a multiple of 8 is 16-byte aligned in x and 8-byte aligned in
// q whatever the row length: rows of odd length move by whole vectors too, all
// but the one or two that a row shares with its neighbours.

#include "common.cuh"

namespace {

constexpr int kWarps = 24;
constexpr int kThreads = kWarps * 32;
constexpr int kSlots = 18;  // vectors of 8 elements that a lane's queue holds
static_assert(kWarps % 8 == 0 && kWarps / 2 < 16, "groups of two warps have a barrier each, of 15");
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, half to even

// Largest |x| of each FP16 half, NaN if one is.
__device__ __forceinline__ __half2 largest(uint4 v, __half2 m) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
  for (int e = 0; e < 4; ++e) m = __hmax2_nan(m, __habs2(h[e]));
  return m;
}

// round_half_even(x / s) from the approximate quotient's rounding q, off by
// at most one. r = x - q s is exact: x and s are multiples of s's last place
// (|x| >= s / 2 here and x has 11 bits to s's 24) and |r| < s.
__device__ __forceinline__ float settle(float x, float s, float q) {
  const float r = fmaf(-q, s, x);
  const float twice = 2.0f * fabsf(r);
  const bool odd = (static_cast<int>(q) & 1) != 0;
  return twice > s || (twice == s && odd) ? q + copysignf(1.0f, r) : q;
}

// The low byte of kMagic + n is the integer n in two's complement.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                     __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}

__device__ __noinline__ uint2 quantize_settled(uint4 v, float s, float inv) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  float t[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(h[e]);
    t[2 * e] = kMagic + settle(f.x, s, fmaf(f.x, inv, kMagic) - kMagic);
    t[2 * e + 1] = kMagic + settle(f.y, s, fmaf(f.y, inv, kMagic) - kMagic);
  }
  return make_uint2(low_bytes(t[0], t[1], t[2], t[3]), low_bytes(t[4], t[5], t[6], t[7]));
}

// Eight integers of one vector, a byte each. inv is 1 / s to 2^-23, so the
// quotient lies between x (1 - 2^-21) inv and x (1 + 2^-21) inv, and where
// those two round to the same integer (they are 2^-13 apart at most), so does
// it. Else, about once in 10^4 elements, it is settled exactly.
__device__ __forceinline__ uint2 quantize(uint4 v, float s, float inv) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const float below = inv * (1.0f - 0x1p-21f), above = inv * (1.0f + 0x1p-21f);
  float t[8], u[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(h[e]);
    t[2 * e] = fmaf(f.x, below, kMagic);
    t[2 * e + 1] = fmaf(f.y, below, kMagic);
    u[2 * e] = fmaf(f.x, above, kMagic);
    u[2 * e + 1] = fmaf(f.y, above, kMagic);
  }
  const uint2 a = make_uint2(low_bytes(t[0], t[1], t[2], t[3]), low_bytes(t[4], t[5], t[6], t[7]));
  const uint2 b = make_uint2(low_bytes(u[0], u[1], u[2], u[3]), low_bytes(u[4], u[5], u[6], u[7]));
  return ((a.x ^ b.x) | (a.y ^ b.y)) == 0 ? a : quantize_settled(v, s, inv);
}

// A row as vectors of 8 elements from the multiple of 8 at or before its
// first one; `head` elements of the first vector and those of the last one
// from `tail` on are not the row's.
struct Row {
  const uint4* x;
  uint2* q;
  int vectors, head, tail;
};

// Vector i without the elements that are not the row's.
__device__ __forceinline__ uint4 trimmed(const Row& r, int i, uint4 v) {
  const int lo = i == 0 ? r.head : 0, hi = i == r.vectors - 1 ? r.tail : 8;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e < lo || e >= hi) w[e / 2] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
  }
  return v;
}

// The row's elements of vector i, written one by one.
__device__ __forceinline__ void store_elements(const Row& r, int i, uint2 w) {
  const int lo = i == 0 ? r.head : 0, hi = i == r.vectors - 1 ? r.tail : 8;
  signed char* q = reinterpret_cast<signed char*>(r.q + i);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e >= lo && e < hi) q[e] = static_cast<signed char>((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
  }
}

// Copies one vector to shared memory: its first `bytes` bytes, zeros for the rest.
__device__ __forceinline__ void copy_vector(uint32_t dst, const uint4* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint4 read_vector(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src)
               : "memory");
  return v;
}

// The maximum of a row over the `warps` warps from `first` on, which meet at
// `barrier` (1 to 15).
__device__ __forceinline__ uint32_t row_maximum(uint32_t m, int first, int warps, int barrier, uint32_t* shared) {
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if (warps > 1) {
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(32 * warps) : "memory");  // the last row's readers are done
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x / 32] = m;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(32 * warps) : "memory");
    for (int w = 0; w < warps; ++w) m = max(m, shared[first + w]);
  }
  return m;
}

// fl32(amax / 127) for FP16 amax: the product with fl32(1 / 127) corrected by
// its exact remainder, which rounds as the division does (P. Markstein, 1990).
__device__ __forceinline__ float scale_of(float amax) {
  const float inverse = 1.0f / 127.0f;
  const float s = amax * inverse;
  return amax < INFINITY ? fmaf(fmaf(-s, 127.0f, amax), inverse, s) : amax;
}

__device__ __forceinline__ Row row_at(const unsigned short* x, signed char* q, long long row, int columns) {
  const long long begin = row * columns, first = begin & ~7ll;
  Row r;
  r.x = reinterpret_cast<const uint4*>(x + first);
  r.q = reinterpret_cast<uint2*>(q + first);
  r.head = static_cast<int>(begin - first);
  r.vectors = (r.head + columns + 7) >> 3;
  r.tail = r.head + columns - 8 * (r.vectors - 1);
  return r;
}

// Batches of `batch` rows of `slots` vectors a lane, kAhead batches in the
// queue, by groups of 2^kWarpsLog2 warps (with the number of warps known to the
// compiler 16384x8192 takes 67 us instead of 75).
template <int kWarpsLog2, int kAhead>
__device__ __forceinline__ void quantize_rows(uint8_t* smem, const unsigned short* x,
                                              signed char* q, float* scale, int rows,
                                              int columns, int slots, int batch, uint32_t* shared) {
  constexpr int kGroupWarps = 1 << kWarpsLog2, kLanesLog2 = 5 + kWarpsLog2, kLanes = 1 << kLanesLog2;
  const int group_in_block = threadIdx.x >> kLanesLog2;
  const int lane = threadIdx.x & (kLanes - 1);
  constexpr int groups_a_block = kWarps >> kWarpsLog2;
  if (kWarps % kGroupWarps != 0 && group_in_block >= groups_a_block) return;  // sixteen warps: eight are left over
  const long long groups = static_cast<long long>(gridDim.x) * groups_a_block;
  const long long group = static_cast<long long>(blockIdx.x) * groups_a_block + group_in_block;
  const long long total = static_cast<long long>(rows) * columns;
  const uint32_t queue = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + (threadIdx.x / 32) * (kSlots * 512) +
                         (threadIdx.x & 31) * 16;
  const uint32_t batch_bytes = static_cast<uint32_t>(batch * slots) * 512;

  long long fetch = group * batch;  // first row of the next batch to copy
  int place = 0;                    // of the next batch in the queue
  const auto copy_batch = [&]() {
    for (int k = 0; k < batch && fetch + k < rows; ++k) {
      const Row r = row_at(x, q, fetch + k, columns);
      // The tensor's last vector may end past it.
      const long long end = (fetch + k) * columns - r.head + 8ll * r.vectors;
      const int last_bytes = end > total ? 16 - 2 * static_cast<int>(end - total) : 16;
      const uint32_t dst = queue + place * batch_bytes + static_cast<uint32_t>(k * slots) * 512;
      const int mine = lane < r.vectors ? ((r.vectors - lane - 1) >> kLanesLog2) + 1 : 0;
#pragma unroll 4
      for (int j = 0; j < mine; ++j) {
        const int i = (j << kLanesLog2) + lane;
        copy_vector(dst + j * 512, r.x + i, i == r.vectors - 1 ? last_bytes : 16);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    fetch += groups * batch;
    place = place + 1 == kAhead ? 0 : place + 1;
  };
#pragma unroll
  for (int a = 0; a < kAhead; ++a) copy_batch();

  int at = 0;
  for (long long row0 = group * batch; row0 < rows; row0 += groups * batch) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    for (int k = 0; k < batch && row0 + k < rows; ++k) {
      const Row r = row_at(x, q, row0 + k, columns);
      const bool ragged = r.head != 0 || r.tail != 8;
      const uint32_t src = queue + at * batch_bytes + static_cast<uint32_t>(k * slots) * 512;
      __half2 pair = __half2half2(__ushort_as_half(0));
      const int mine = lane < r.vectors ? ((r.vectors - lane - 1) >> kLanesLog2) + 1 : 0;
#pragma unroll 4
      for (int j = 0; j < mine; ++j) {
        const int i = (j << kLanesLog2) + lane;
        uint4 v = read_vector(src + j * 512);
        if (ragged && (i == 0 || i == r.vectors - 1)) v = trimmed(r, i, v);
        pair = largest(v, pair);
      }
      const uint32_t bits = *reinterpret_cast<uint32_t*>(&pair) & 0x7FFF7FFFu;
      const uint32_t m = row_maximum(max(bits & 0xFFFFu, bits >> 16), group_in_block << kWarpsLog2, kGroupWarps,
                                     1 + group_in_block, shared);
      const float s = scale_of(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
      if (lane == 0) scale[row0 + k] = s;
      float inv;
      asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
      const bool regular = m != 0 && m < 0x7C00u;
#pragma unroll 4
      for (int j = 0; j < mine; ++j) {
        const int i = (j << kLanesLog2) + lane;
        const uint2 packed = regular ? quantize(read_vector(src + j * 512), s, inv) : make_uint2(0, 0);
        if (ragged && (i == 0 || i == r.vectors - 1)) {
          store_elements(r, i, packed);
        } else {
          r.q[i] = packed;
        }
      }
    }
    at = at + 1 == kAhead ? 0 : at + 1;
    // The batch's last values are in registers: its place may be overwritten.
    copy_batch();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// One row by a block, element by element: tensors off 16 bytes (x) or 8 (q), and
// rows longer than the queues of sixteen warps.
__device__ __forceinline__ void quantize_row_unaligned(const unsigned short* x, signed char* q, float* scale,
                                                       long long row, int columns, uint32_t* shared) {
  const unsigned short* xr = x + row * columns;
  uint32_t m = 0;
  for (int i = threadIdx.x; i < columns; i += kThreads) m = max(m, static_cast<uint32_t>(xr[i]) & 0x7FFFu);
  m = row_maximum(m, 0, kWarps, 1, shared);
  const float s = scale_of(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
  if (threadIdx.x == 0) scale[row] = s;
  const bool regular = m != 0 && m < 0x7C00u;
  const float inv = regular ? __frcp_rn(s) : 0.0f;
  // Four loads before four stores: x may not be read through the read-only path
  // (its writer can still run when this grid starts), so the compiler keeps
  // every load behind the stores in front of it.
  const unsigned n = static_cast<unsigned>(columns);
  for (unsigned i0 = threadIdx.x; i0 < n; i0 += 4 * kThreads) {
    unsigned short v[4];
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) v[j] = i0 + j * kThreads < n ? xr[i0 + j * kThreads] : 0;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const unsigned i = i0 + j * kThreads;
      const float f = __half2float(__ushort_as_half(v[j]));
      if (i < n) q[row * columns + i] = regular ? static_cast<signed char>(settle(f, s, rintf(f * inv))) : 0;
    }
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads, 1)
ctb_quantize_rows_f16(const unsigned short* x, signed char* q, float* scale, int rows, int columns,
                      CTB_RESERVED_PARAMS) {
  CTB_UNUSED_RESERVED();
  CTB_GRID_DEPENDENCY_SYNC();
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* shared = reinterpret_cast<uint32_t*>(smem + kWarps * kSlots * 512);
  // At most: a row of a length that 8 does not divide may begin inside a vector.
  const int vectors = columns % 8 == 0 ? columns / 8 : (columns + 14) / 8;
  if (!ctb::aligned16(x) || (reinterpret_cast<uintptr_t>(q) & 7u) != 0 || vectors > 16 * 32 * kSlots) {
    for (int row = blockIdx.x; row < rows; row += gridDim.x) quantize_row_unaligned(x, q, scale, row, columns, shared);
    return;
  }
  // Warps a row: those that finish first, by rounds of rows over the groups of
  // warps and a row's slots plus two for its maximum, among those whose queues
  // hold two rows (eight and sixteen warps: one). 16384 rows of 2048: one warp
  // 22 us, two 24; 2048 rows of 4096: four 9.0 us, two 10.5; 8 rows of 12288:
  // sixteen 2.9 us, eight 4.4 us; 2048 rows of 40000: sixteen 65 us, element by
  // element 232 us.
  // Lane w rates 2^w warps; ties go to the most.
  const int w = min(static_cast<int>(threadIdx.x & 31), 4);
  const int lane_vectors = (vectors + (32 << w) - 1) >> (5 + w);
  const float turns = ceilf(__fdividef(static_cast<float>(rows), static_cast<float>(gridDim.x * (kWarps >> w))));
  const unsigned cost = static_cast<unsigned>(fminf(turns * static_cast<float>(lane_vectors + 2), 4e8f));
  const unsigned rated = lane_vectors <= (w >= 3 ? kSlots : kSlots / 2) ? cost * 8u + static_cast<unsigned>(4 - w) : ~0u;
  const int warps_log2 = 4 - static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, rated) & 7u);
  const int slots = (vectors + (32 << warps_log2) - 1) >> (5 + warps_log2);
  const int rounds = static_cast<int>(__shfl_sync(0xFFFFFFFFu, turns, warps_log2));
  if (warps_log2 == 0 && slots <= kSlots / 4) {
    quantize_rows<0, 4>(smem, x, q, scale, rows, columns, slots,
                         min(rounds, kSlots / 4 / slots), shared);
  } else if (warps_log2 == 0) {
    quantize_rows<0, 2>(smem, x, q, scale, rows, columns, slots, 1, shared);
  } else if (warps_log2 == 1) {
    quantize_rows<1, 2>(smem, x, q, scale, rows, columns, slots, 1, shared);
  } else if (warps_log2 == 2) {
    quantize_rows<2, 2>(smem, x, q, scale, rows, columns, slots, 1, shared);
  } else if (warps_log2 == 3 && slots <= kSlots / 2) {
    quantize_rows<3, 2>(smem, x, q, scale, rows, columns, slots, 1, shared);
  } else if (warps_log2 == 3) {
    quantize_rows<3, 1>(smem, x, q, scale, rows, columns, slots, 1, shared);
  } else if (slots <= kSlots / 2) {
    quantize_rows<4, 2>(smem, x, q, scale, rows, columns, slots, 1, shared);
  } else {
    quantize_rows<4, 1>(smem, x, q, scale, rows, columns, slots, 1, shared);
  }
}
