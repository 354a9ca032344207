// GatedGemm, QGemm and QGatedGemm for few rows (at most 16): the weights pass
// once from HBM through every SM, and nothing else costs time.
//
// With M rows each weight takes part in M multiply-adds, so here the product is
// bound by reading the weights (K N elements, twice for the gated
// ops). What that needs is every SM reading at the same rate to the end and
// enough bytes in flight (about 45 KB an SM), not tensor throughput:
//
// * One CTA an SM; the CTAs share the output columns out evenly in groups of
//   8. The reading warps of a CTA take the 64-byte chunks of K in turn. A batch
//   is four groups of weight rows, for the gated ops four of each matrix.
// * A warp reads a batch's chunk of 8 rows x 64 bytes with one 16-byte
//   cp.async a lane into a queue in shared memory that is private to the
//   lane, so the copies need no barrier: a lane waits for its own oldest
//   group, reads its own 16 bytes back and refills the slot. The queue runs
//   on over batches.
// * The lane's 16 bytes are its operand of mma.sync as they lie: lane (g, q)
//   holds row g and k 8 q .. 8 q + 7 (16 q .. in 8 bits) of the chunk, words
//   {0, 1} serve as the fragment of one MMA and {2, 3} of the next. That
//   permutes k within a chunk, and x is loaded with the same permutation
//   through the same queue (from L2, where it stays).
// * Four further warps join a batch's sums over the readers, in a fixed order
//   (results do not depend on timing), and store the outputs. The join buffer
//   is double, so no reading warp waits for another one: when all of them met
//   at a barrier after each batch (joined over a cluster of two CTAs, K split
//   in 16), 16x4096x12288 took 24 % longer and the 8-bit form for 8 rows 42 %.
// 16x4096x12288 takes 37.0 us, in 8 bits 21.2 and 20.4 for 8 rows;
// 1x4096x12288 reads its 201 MB in 34.8 us, 5.8 TB/s.
// All waits are bounded (tc_common.cuh).

#include "product.cuh"
#include "tc_common.cuh"

namespace {

using ctb::tc::mbar_arrive;
using ctb::tc::mbar_init;
using ctb::tc::mbar_wait;

constexpr int kJoinWarps = 4;
// Threads of a block: the most reading warps of a form and the joining ones.
constexpr int kPlainThreads = (16 + kJoinWarps) * 32;
constexpr int kGatedThreads = (12 + kJoinWarps) * 32;
constexpr int kSharedBytes = 231424;  // barriers, join buffers, queues

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
  void* scratch;
};

struct Barriers {
  uint64_t full[2];   // the reading warps have left their sums in a join buffer
  uint64_t empty[2];  // the joining warps have read it
  int abort;
};

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

// kTokens8: groups of 8 rows of x (1 or 2). kWarps: reading warps, over which K
// is split.
template <typename T, bool kGated, int kTokens8, int kWarps>
__device__ __forceinline__ void product_stream(uint8_t* smem, const Operands<T>& op) {
  using Sum = typename T::Sum;
  constexpr int kGroups = kGated ? 8 : 4;     // groups of 8 weight rows a batch
  constexpr int kStride = 8 * kGroups + 8;    // words a token in the join buffer (conflict-free pairs)
  constexpr int kPieces = kGroups + kTokens8;  // 16-byte pieces a lane and slot
  constexpr int kSlotBytes = kPieces * 512;    // a warp's
  constexpr int kTokens = 8 * kTokens8;
  constexpr int kJoin = kWarps * kTokens * kStride;  // words a join buffer
  constexpr int kDepth = (kSharedBytes - 128 - 8 * kJoin) / (kWarps * kSlotBytes);
  static_assert(kDepth >= 3, "queue");
  constexpr int kMTiles = (kTokens8 + 1) / 2;
  constexpr int kChannelGroups = 4;  // output groups a batch
  constexpr int kChunk = 4 * T::kPiece;

  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const long long groups = (static_cast<long long>(op.n) + 7) / 8;
  const long long first = groups * blockIdx.x / gridDim.x, last = groups * (blockIdx.x + 1) / gridDim.x;
  const int batches = static_cast<int>((last - first + kChannelGroups - 1) / kChannelGroups);

  Barriers* bars = reinterpret_cast<Barriers*>(smem);
  volatile int* abort = &bars->abort;
  Sum* join = reinterpret_cast<Sum*>(smem + 128);
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->full[b], kWarps);
      mbar_init(&bars->empty[b], kJoinWarps);
    }
    bars->abort = 0;
    ctb::tc::mbar_init_fence();
  }
  __syncthreads();

  if (warp < kWarps) {
    // ---- reading warps: chunks `warp`, `warp` + kWarps, ... of K ----
    const int g = lane >> 2, q = lane & 3;
    const int chunks = (op.k + kChunk - 1) / kChunk;
    const int mine = chunks > warp ? (chunks - warp - 1) / kWarps + 1 : 0;
    const uint32_t queue = ctb::tc::smem_addr(smem + 128 + 8 * kJoin) + warp * (kDepth * kSlotBytes) + lane * 16;

    // The (batch, chunk) that the next refill takes.
    int fill_batch = 0, fill_chunk = 0;
    const typename T::Element* rows[kGroups];
    int row_bytes[kGroups];
    const auto set_rows = [&]() {
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        const long long group = first + fill_batch * kChannelGroups + i % kChannelGroups;
        const long long row = group * 8 + g;
        const bool inside = group < last && row < op.n;
        const auto* w = kGated && i >= kChannelGroups ? op.w[1] : op.w[0];
        rows[i] = inside ? w + row * op.k : w;
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
        const int k0 = (warp + kWarps * fill_chunk) * kChunk + q * T::kPiece;
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
      const int buffer = batch & 1;
      if (batch >= 2 && !mbar_wait(&bars->empty[buffer], ((batch >> 1) - 1) & 1, abort, op.scratch, 81)) break;
#pragma unroll
      for (int t = 0; t < kMTiles; ++t)
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          Sum* dst = join + buffer * kJoin + (warp * kTokens + 16 * t + g) * kStride + 8 * i + 2 * q;
          dst[0] = sum[t][i][0];
          dst[1] = sum[t][i][1];
          if (2 * t + 1 < kTokens8) {
            dst[8 * kStride] = sum[t][i][2];
            dst[8 * kStride + 1] = sum[t][i][3];
          }
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->full[buffer]);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    return;
  }

  if (warp >= kWarps + kJoinWarps) return;

  // ---- joining warps: tokens j, j + 4, ...; lane = output column of the batch ----
  const int j = warp - kWarps;
  for (int batch = 0; batch < batches; ++batch) {
    const int buffer = batch & 1;
    const bool ready = mbar_wait(&bars->full[buffer], (batch >> 1) & 1, abort, op.scratch, 82);
    __syncwarp();
    if (!ready) break;
    Sum total[kTokens / kJoinWarps], up[kTokens / kJoinWarps];
#pragma unroll
    for (int r = 0; r < kTokens / kJoinWarps; ++r) {
      const int token = j + kJoinWarps * r;
      total[r] = up[r] = 0;
      if (token >= op.m) continue;
      const Sum* src = join + buffer * kJoin + token * kStride + lane;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        total[r] += src[v * kTokens * kStride];
        if (kGated) up[r] += src[v * kTokens * kStride + 32];
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->empty[buffer]);
    const long long column = (first + batch * kChannelGroups) * 8 + lane;
    if (column >= op.n || column >= last * 8) continue;
    float scale = 0.0f, up_scale = 0.0f, bias = 0.0f;
    if (T::kPiece == 16) {
      scale = op.w_scale[0][column];
      if (kGated) up_scale = op.w_scale[1][column];
      if (!kGated && op.bias != nullptr) bias = __half2float(op.bias[column]);
    }
#pragma unroll
    for (int r = 0; r < kTokens / kJoinWarps; ++r) {
      const int token = j + kJoinWarps * r;
      if (token >= op.m) continue;
      float y = static_cast<float>(total[r]), u = static_cast<float>(up[r]);
      if constexpr (T::kPiece == 16) {
        const float row_scale = op.x_scale[token];
        y = ctb::dequantized(total[r], row_scale, scale, bias);
        if (kGated) u = ctb::dequantized(up[r], row_scale, up_scale, 0.0f);
      }
      if (kGated) y = ctb::gated(y, u, op.activation);
      op.out[static_cast<long long>(token) * op.n + column] = __float2half_rn(y);
    }
  }
}

template <typename T, bool kGated>
__device__ __forceinline__ void product_dispatch(const Operands<T>& op) {
  extern __shared__ __align__(16) uint8_t smem[];
  // More rows, rows of x or of weights off 16 bytes: not this kernel's (the
  // host offers it only for the rest; a tensor bound off 16 bytes ends here).
  bool fits = op.m <= 16 && op.k % T::kPiece == 0 && ctb::aligned16(op.x) && ctb::aligned16(op.w[0]);
  if (kGated) fits = fits && ctb::aligned16(op.w[1]);
  if (!fits) {
    if (threadIdx.x == 0) ctb::report_error(op.scratch, ctb::kErrorBadShape, 80);
    return;
  }
  // Reading warps: as many as leave every queue three slots and more beside
  // the join buffers (16x4096x12288 with twelve 25 % longer).
  constexpr int kFew = kGated ? 12 : 16, kMore = kGated ? 8 : 16;
  if (op.m <= 8) {
    product_stream<T, kGated, 1, kFew>(smem, op);
  } else {
    product_stream<T, kGated, 2, kMore>(smem, op);
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kGatedThreads, 1)
ctb_gated_gemm_f16_stream(const __half* x, const __half* w_gate, const __half* w_up, __half* output, int m, int n,
                          int k, int activation, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  CTB_GRID_DEPENDENCY_SYNC();
  const Operands<Half> op = {x, {w_gate, w_up}, nullptr, {nullptr, nullptr}, nullptr, output, m, n, k, activation, runtime_scratch};
  product_dispatch<Half, true>(op);
}

extern "C" __global__ void __launch_bounds__(kPlainThreads, 1)
ctb_qgemm_i8_stream(const signed char* x, const signed char* w, const float* x_scale, const float* w_scale,
                    const __half* bias, __half* output, int m, int n, int k, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  CTB_GRID_DEPENDENCY_SYNC();
  const Operands<Int8> op = {x, {w, nullptr}, x_scale, {w_scale, nullptr}, bias, output, m, n, k, 0, runtime_scratch};
  product_dispatch<Int8, false>(op);
}

extern "C" __global__ void __launch_bounds__(kGatedThreads, 1)
ctb_qgated_gemm_i8_stream(const signed char* x, const signed char* w_gate, const signed char* w_up,
                          const float* x_scale, const float* gate_scale, const float* up_scale, __half* output, int m,
                          int n, int k, int activation, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  CTB_GRID_DEPENDENCY_SYNC();
  const Operands<Int8> op = {x, {w_gate, w_up}, x_scale, {gate_scale, up_scale}, nullptr, output, m, n, k, activation, runtime_scratch};
  product_dispatch<Int8, true>(op);
}
