// GatedGemm, QGemm and QGatedGemm for few rows (at most 32): the weights pass
// once from HBM through every SM, and nothing else costs time.
//
// With M rows each weight takes part in M multiply-adds, so up to M = 32 the
// product is bound by reading the weights (K N elements, twice for the gated
// ops). What that needs is every SM reading at the same rate to the end and
// enough bytes in flight (about 45 KB an SM), not tensor throughput:
//
// * Clusters of two CTAs (one a SM) share the output columns out evenly in
//   groups of 8, so that their loads differ by one group at most, and each of
//   the cluster's 16 warps takes every 16th 64-byte chunk of K. A batch is four
//   groups of weight rows (for the gated ops two of each matrix).
// * A warp reads a batch's chunk of 8 rows x 64 bytes with one 16-byte
//   cp.async a lane into a queue in shared memory that is private to the
//   lane, so the copies need no barrier: a lane waits for its own oldest
//   group, reads its own 16 bytes back and refills the slot. The queue runs
//   on over batches; 5 to 8 slots of 2 KB a warp keep 80 to 128 KB in flight.
// * The lane's 16 bytes are its operand of mma.sync as they lie: lane (g, q)
//   holds row g and k 8 q .. 8 q + 7 (16 q .. in 8 bits) of the chunk, words
//   {0, 1} serve as the fragment of one MMA and {2, 3} of the next. That
//   permutes k within a chunk, and x is loaded with the same permutation
//   through the same queue (from L2, where it stays).
// * A batch's sums are joined over the CTA's 8 warps in shared memory and over
//   the two CTAs by remote stores, in a fixed order: results do not depend on
//   timing. One cluster barrier a batch, hidden behind the queue.
//
// No loop waits on memory that another thread writes: the only waits are
// cp.async groups and hardware barriers that every thread reaches.

#include "product.cuh"

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kSplit = 2 * kWarps;  // warps of the cluster, over which K is split
constexpr int kGroups = 4;          // groups of 8 weight rows a batch
constexpr int kStride = 40;         // words a token in the join buffer (conflict-free pairs)
constexpr int kQueueBytes = 180224;
constexpr int kJoinBytes = kWarps * 32 * kStride * 4;  // 32 tokens
constexpr int kRemoteBytes = 2 * 32 * 32 * 4;

struct Half {
  using Element = __half;
  using Sum = float;
  static constexpr int kPiece = 8;  // elements of 16 bytes
  static __device__ __forceinline__ void mma(Sum (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
struct Int8 {
  using Element = signed char;
  using Sum = int;
  static constexpr int kPiece = 16;
  static __device__ __forceinline__ void mma(Sum (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

template <typename T>
struct Operands {
  const typename T::Element* x;
  const typename T::Element* w[2];
  const float* x_scale;
  const float* w_scale[2];
  const __half* bias;
  __half* out;
  int m, n, k, activation;
};

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes, or 16 zero bytes when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint4 read_16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src)
               : "memory");
  return v;
}

// kTokens8: groups of 8 rows of x (1, 2 or 4).
template <typename T, bool kGated, int kTokens8>
__device__ __forceinline__ void product_stream(uint8_t* smem, const Operands<T>& op) {
  using Sum = typename T::Sum;
  constexpr int kPieces = kGroups + kTokens8;           // 16-byte pieces a lane and slot
  constexpr int kSlotBytes = kPieces * 512;             // a warp's
  constexpr int kDepth = kQueueBytes / (kWarps * kSlotBytes);
  constexpr int kMTiles = (kTokens8 + 1) / 2;
  constexpr int kChannelGroups = kGated ? kGroups / 2 : kGroups;  // output groups a batch
  constexpr int kChunk = 4 * T::kPiece;

  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int cluster = blockIdx.x / 2, clusters = gridDim.x / 2;
  const long long groups = (op.n + 7) / 8;
  const int first = static_cast<int>(groups * cluster / clusters);
  const int last = static_cast<int>(groups * (cluster + 1) / clusters);
  const int batches = (last - first + kChannelGroups - 1) / kChannelGroups;

  // This warp's chunks of K: `at`, `at` + 16, ...
  const int at = static_cast<int>(rank) * kWarps + warp;
  const int chunks = (op.k + kChunk - 1) / kChunk;
  const int mine = chunks > at ? (chunks - at - 1) / kSplit + 1 : 0;

  const uint32_t queue = shared_addr(smem) + warp * (kDepth * kSlotBytes) + lane * 16;
  Sum* join = reinterpret_cast<Sum*>(smem + kQueueBytes);
  Sum* remote = reinterpret_cast<Sum*>(smem + kQueueBytes + kJoinBytes);
  uint32_t peer_remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer_remote) : "r"(shared_addr(remote)), "r"(rank ^ 1u));

  // The peer's shared memory exists from here on (waited for below).
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  // ---- producer: the (batch, chunk) the next refill takes ----
  int fill_batch = 0, fill_chunk = 0;
  const typename T::Element* rows[kGroups];
  int row_bytes[kGroups];
  const auto set_rows = [&]() {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int group = first + fill_batch * kChannelGroups + i % kChannelGroups;
      const int row = group * 8 + g;
      const bool inside = group < last && row < op.n;
      const auto* w = kGated && i >= kChannelGroups ? op.w[1] : op.w[0];
      rows[i] = inside ? w + static_cast<long long>(row) * op.k : w;
      row_bytes[i] = inside ? 16 : 0;
    }
  };
  const typename T::Element* tokens[kTokens8];
  int token_bytes[kTokens8];
#pragma unroll
  for (int r = 0; r < kTokens8; ++r) {
    const bool inside = r * 8 + g < op.m;
    tokens[r] = inside ? op.x + static_cast<long long>(r * 8 + g) * op.k : op.x;
    token_bytes[r] = inside ? 16 : 0;
  }
  set_rows();
  const auto refill = [&](int slot) {
    if (fill_batch < batches && mine > 0) {
      const int k0 = (at + kSplit * fill_chunk) * kChunk + q * T::kPiece;
      const bool inside = k0 < op.k;  // K is a multiple of a piece
      const int offset = inside ? k0 : 0;
      const uint32_t dst = queue + slot * kSlotBytes;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) copy_16(dst + i * 512, rows[i] + offset, inside ? row_bytes[i] : 0);
#pragma unroll
      for (int r = 0; r < kTokens8; ++r) {
        copy_16(dst + (kGroups + r) * 512, tokens[r] + offset, inside ? token_bytes[r] : 0);
      }
      if (++fill_chunk == mine) {
        fill_chunk = 0;
        ++fill_batch;
        set_rows();
      }
    }
    // A group is committed even when it is empty: slots are counted by groups.
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kDepth; ++s) refill(s);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  int slot = 0;
  for (int batch = 0; batch < batches; ++batch) {
    Sum sum[kMTiles][kGroups][4];
#pragma unroll
    for (int t = 0; t < kMTiles; ++t)
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[t][i][j] = 0;
    for (int c = 0; c < mine; ++c) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      const uint32_t src = queue + slot * kSlotBytes;
      uint4 w[kGroups], x[2 * kMTiles];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) w[i] = read_16(src + i * 512);
#pragma unroll
      for (int r = 0; r < 2 * kMTiles; ++r) {
        x[r] = r < kTokens8 ? read_16(src + (kGroups + r) * 512) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < kMTiles; ++t) {
        const uint4 a = x[2 * t], b = x[2 * t + 1];
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          T::mma(sum[t][i], a.x, b.x, a.y, b.y, w[i].x, w[i].y);
          T::mma(sum[t][i], a.z, b.z, a.w, b.w, w[i].z, w[i].w);
        }
      }
      // The MMAs have taken the slot's values: it may be overwritten.
      refill(slot);
      slot = slot + 1 == kDepth ? 0 : slot + 1;
    }
    // ---- join: 8 warps, then 2 CTAs ----
#pragma unroll
    for (int t = 0; t < kMTiles; ++t)
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        Sum* dst = join + (warp * (8 * kTokens8) + 16 * t + g) * kStride + 8 * i + 2 * q;
        dst[0] = sum[t][i][0];
        dst[1] = sum[t][i][1];
        if (2 * t + 1 < kTokens8) {
          dst[8 * kStride] = sum[t][i][2];
          dst[8 * kStride + 1] = sum[t][i][3];
        }
      }
    __syncthreads();
    // Warp w has tokens w, w + 8, ...; lane = column of the batch. CTA 0
    // finishes the even tokens, CTA 1 the odd ones.
    const bool owner = (warp & 1) == static_cast<int>(rank);
    Sum total[kTokens8];
    const int buffer = (batch & 1) * (8 * kTokens8 * 32);
#pragma unroll
    for (int r = 0; r < kTokens8; ++r) {
      const int token = warp + 8 * r;
      if (token >= op.m) continue;
      Sum s = 0;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) s += join[(v * (8 * kTokens8) + token) * kStride + lane];
      total[r] = s;
      if (!owner) {
        const uint32_t dst = peer_remote + (buffer + token * 32 + lane) * 4;
        uint32_t bits;
        memcpy(&bits, &s, 4);
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(bits) : "memory");
      }
    }
    // Also the barrier between this batch's reads of `join` and the next
    // one's writes; `remote` alternates between two buffers.
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (!owner) continue;
    const int group0 = first + batch * kChannelGroups;
    const int column = group0 * 8 + (kGated ? lane & 15 : lane);
    const bool inside = column < op.n && column < last * 8;
    float column_scale = 0.0f, bias = 0.0f;
    if (T::kPiece == 16 && inside) {
      column_scale = __ldg((kGated && lane >= 16 ? op.w_scale[1] : op.w_scale[0]) + column);
      if (!kGated && op.bias != nullptr) bias = __half2float(op.bias[column]);
    }
#pragma unroll
    for (int r = 0; r < kTokens8; ++r) {
      const int token = warp + 8 * r;
      if (token >= op.m) continue;
      const Sum s = total[r] + remote[buffer + token * 32 + lane];
      float y = static_cast<float>(s);
      if constexpr (T::kPiece == 16) {
        y = ctb::dequantized(s, __ldg(op.x_scale + token), column_scale, bias);
      }
      if constexpr (kGated) {
        const float up = __shfl_down_sync(0xFFFFFFFFu, y, 16);
        y = ctb::gated(y, up, op.activation);
        if (lane >= 16) continue;
      }
      if (inside) op.out[static_cast<long long>(token) * op.n + column] = __float2half_rn(y);
    }
  }
}

template <typename T, bool kGated>
__device__ __forceinline__ void product_dispatch(const Operands<T>& op, void* scratch) {
  extern __shared__ __align__(16) uint8_t smem[];
  static_assert(kQueueBytes + kJoinBytes + kRemoteBytes <= 232448, "shared memory");
  // More rows, rows of x or of weights off 16 bytes: not this kernel's (the
  // host offers it only for the rest; a tensor bound off 16 bytes ends here).
  bool fits = op.m <= 32 && op.k % T::kPiece == 0 && ctb::aligned16(op.x) && ctb::aligned16(op.w[0]);
  if (kGated) fits = fits && ctb::aligned16(op.w[1]);
  if (!fits) {
    if (threadIdx.x == 0) ctb::report_error(scratch, ctb::kErrorBadShape, 80);
    return;
  }
  if (op.m <= 8) {
    product_stream<T, kGated, 1>(smem, op);
  } else if (op.m <= 16) {
    product_stream<T, kGated, 2>(smem, op);
  } else {
    product_stream<T, kGated, 4>(smem, op);
  }
}

}  // namespace

extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ctb_gated_gemm_f16_stream(const __half* x, const __half* w_gate, const __half* w_up, __half* output, int m, int n,
                          int k, int activation, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  CTB_GRID_DEPENDENCY_SYNC();
  const Operands<Half> op = {x, {w_gate, w_up}, nullptr, {nullptr, nullptr}, nullptr, output, m, n, k, activation};
  product_dispatch<Half, true>(op, runtime_scratch);
}

extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ctb_qgemm_i8_stream(const signed char* x, const signed char* w, const float* x_scale, const float* w_scale,
                    const __half* bias, __half* output, int m, int n, int k, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  CTB_GRID_DEPENDENCY_SYNC();
  const Operands<Int8> op = {x, {w, nullptr}, x_scale, {w_scale, nullptr}, bias, output, m, n, k, 0};
  product_dispatch<Int8, false>(op, runtime_scratch);
}

extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ctb_qgated_gemm_i8_stream(const signed char* x, const signed char* w_gate, const signed char* w_up,
                          const float* x_scale, const float* gate_scale, const float* up_scale, __half* output, int m,
                          int n, int k, int activation, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  CTB_GRID_DEPENDENCY_SYNC();
  const Operands<Int8> op = {x, {w_gate, w_up}, x_scale, {gate_scale, up_scale}, nullptr, output, m, n, k, activation};
  product_dispatch<Int8, true>(op, runtime_scratch);
}
