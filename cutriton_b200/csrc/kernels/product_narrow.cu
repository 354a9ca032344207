// GatedGemm, QGemm and QGatedGemm for 17 to 32 rows, QGemm to 64 (tcgen05,
// weights as the left operand).
//
// With so few rows the product is bound by reading the weights, but a tile with
// x on its M side pads 32 rows to 128 and more, and its MMAs take as long as the
// weights take to arrive. So here the weight rows are the M side (128 output
// channels a CTA, of gate and of up for the gated ops) and the rows of x the N
// side: a block of 128 bytes of K costs 64 to 128 clocks of MMAs and brings 4 or
// 8 KB of x beside 16 or 32 KB of weights. 32x4096x12288 gated: 35.9 us, 5.6
// TB/s, for 42.8 by CTA pairs; 8-bit 32x8192x28672 gated 78 us, 6.0 TB/s, for 93.
//
// K is split over the kSplit CTAs of a cluster, so that narrow outputs occupy
// every SM too. Each CTA leaves its sums [token][channel] in its own shared
// memory and joins a share of the tokens over the cluster, in a fixed order
// (results do not depend on timing), four channels a thread (with one a thread
// 4 % more). Two CTAs share an SM: one starts or joins while the other one reads.
//
// TMEM is allocated between the dependency wait and the launch of dependents:
// a CTA that waits for an earlier kernel holds none, and one that a later
// kernel waits for has got its own.
// All waits are bounded (tc_common.cuh).

#include "product.cuh"
#include "tc_common.cuh"

namespace {

using namespace ctb::tc;

constexpr int kChannels = 128;  // weight rows of a matrix a CTA
constexpr int kRowBytes = 128;  // a block of K
constexpr int kThreads = 192;  // loads, MMAs, four epilogue warps
constexpr uint32_t kRingBytes = 110592;
constexpr int kMaxStages = 5;

struct Half {
  static constexpr int kBlock = 64;
  using Sum = float;
  static __host__ __device__ constexpr uint32_t idesc(uint32_t m, uint32_t n) { return instr_desc(kFormatF16, m, n); }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    umma_f16(d, a, b, idesc, accumulate);
  }
  static __device__ __forceinline__ Sum sum(uint32_t bits) { return __uint_as_float(bits); }
};
struct Int8 {
  static constexpr int kBlock = 128;
  using Sum = int;
  // Signed 8-bit operands (format 1), 32-bit integer sums (D format 2).
  static __device__ __forceinline__ uint32_t idesc(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
  static __device__ __forceinline__ Sum sum(uint32_t bits) { return static_cast<int>(bits); }
};

struct __align__(8) Barriers {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t done;  // all MMAs
  uint32_t tmem_base;
  int abort;
};

struct Operands {
  const TmaDescriptor* x32;  // boxes of 32 and 64 rows
  const TmaDescriptor* x64;  // (kMaxTokens = 64)
  const TmaDescriptor* w[2];
  const float* x_scale;
  const float* w_scale[2];
  const __half* bias;
  __half* out;
  int m, n, k, activation;
  void* scratch;
};

__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(elected));
  return elected != 0;
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, void* scratch,
                                          unsigned int site) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort, scratch, site));
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint4 read_cluster(uint32_t local, uint32_t rank) {
  uint32_t remote;
  uint4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(remote)
               : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void add(typename T::Sum (&sum)[4], uint4 v) {
  sum[0] += T::sum(v.x);
  sum[1] += T::sum(v.y);
  sum[2] += T::sum(v.z);
  sum[3] += T::sum(v.w);
}

// kMaxTokens: rows of x that the form takes, 32 or 64.
template <typename T, bool kGated, int kSplit, int kMaxTokens>
__device__ __forceinline__ void product_narrow(const Operands& op) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  Barriers* bars = reinterpret_cast<Barriers*>(smem + kRingBytes);
  volatile int* abort = &bars->abort;
  constexpr int kMatrices = kGated ? 2 : 1;
  static_assert(kMatrices * kMaxTokens * kChannels * 4 <= kRingBytes, "the joined sums lie in the ring");
  constexpr uint32_t kTmemCols = kMatrices * kMaxTokens;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int tokens = kMaxTokens == 32 || op.m <= 32 ? 32 : 64;  // of the MMAs
  const TmaDescriptor* x = tokens == 32 ? op.x32 : op.x64;
  const int x_bytes = tokens * kRowBytes;
  const int stage_bytes = x_bytes + kMatrices * kChannels * kRowBytes;  // a multiple of 1024
  constexpr int kWeightBytes = kMatrices * kChannels * kRowBytes;
  constexpr int kFit32 = kRingBytes / (kWeightBytes + 32 * kRowBytes), kFit64 = kRingBytes / (kWeightBytes + 64 * kRowBytes);
  const int stages = min(kMaxStages, tokens == 32 ? kFit32 : kFit64);
  const int part = static_cast<int>(cluster_rank());
  const int n0 = static_cast<int>(blockIdx.x / kSplit) * kChannels;
  const int k_blocks = (op.k + T::kBlock - 1) / T::kBlock;
  const int first = static_cast<int>(static_cast<long long>(k_blocks) * part / kSplit);
  const int last = static_cast<int>(static_cast<long long>(k_blocks) * (part + 1) / kSplit);
  const int mine = last - first;

  if (warp == 0) {
    if (lane < 2 * kMaxStages) mbar_init(&bars->full[0] + lane, 1);  // full, then empty
    if (lane == 0) {
      mbar_init(&bars->done, 1);
      bars->abort = 0;
    }
    mbar_init_fence();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // More rows are not this kernel's (the host does not offer it for them).
  const bool fits = op.m <= kMaxTokens;

  if (warp == 0 && fits) {
    // ---- loads of this CTA's part of K ----
    int s = 0, issued = 0;
    uint32_t phase = 1;  // the first round of the ring finds every stage free
    for (int kb = first; kb < last; ++kb) {
      if (!warp_wait(&bars->empty[s], phase, abort, op.scratch, 90)) break;
      if (elect_one()) {
        uint8_t* a = smem + s * stage_bytes;
        mbar_arrive_expect_tx(&bars->full[s], stage_bytes);
        tma_load_2d(a, op.w[0], &bars->full[s], kb * T::kBlock, n0);
        if (kGated) tma_load_2d(a + kChannels * kRowBytes, op.w[1], &bars->full[s], kb * T::kBlock, n0);
        tma_load_2d(a + kMatrices * kChannels * kRowBytes, x, &bars->full[s], kb * T::kBlock, 0);
      }
      __syncwarp();
      ++issued;
      if (++s == stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (*abort && lane == 0) {
      // Let the issued copies land before shared memory is released.
      for (int q = max(0, issued - stages); q < issued; ++q) {
        volatile int never = 0;
        mbar_wait(&bars->full[q % stages], (q / stages) & 1, &never, op.scratch, 91);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
  }
  tc_fence_before_sync();
  if (warp != 0) {  // (warp 0 joins at the end)
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  tc_fence_after_sync();
  const uint32_t tmem = warp == 0 ? 0u : *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);

  if (warp == 1 && fits) {
    // ---- MMAs: channels x tokens, one lane issues ----
    const uint32_t idesc = T::idesc(kChannels, tokens);
    const uint64_t first_desc = smem_desc_kmajor_sw128(smem);
    int s = 0;
    uint32_t phase = 0;
    for (int kb = 0; kb < mine; ++kb) {
      if (!warp_wait(&bars->full[s], phase, abort, op.scratch, 92)) break;
      tc_fence_after_sync();
      if (elect_one()) {
        const uint64_t a = first_desc + (static_cast<uint32_t>(s * stage_bytes) >> 4);
        const uint64_t b = a + (kMatrices * kChannels * kRowBytes >> 4);
#pragma unroll
        for (int mat = 0; mat < kMatrices; ++mat)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            T::mma(tmem + mat * kMaxTokens, a + (mat * kChannels * kRowBytes >> 4) + 2 * kk, b + 2 * kk, idesc,
                   (kb | kk) != 0);
          }
        umma_commit(&bars->empty[s]);
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        phase ^= 1;
      }
    }
    // Also after an abandoned wait: what was issued ends before TMEM is freed.
    if (elect_one()) umma_commit(&bars->done);
    __syncwarp();
  }
  uint32_t* sums = reinterpret_cast<uint32_t*>(smem);  // [matrix][token][channel]
  if (warp >= 2 && fits) {
    // ---- this part's sums to shared memory; lane = channel ----
    const int channel = (warp & 3) * 32 + lane;
    const bool ready = warp_wait(&bars->done, 0, abort, op.scratch, 93);
    tc_fence_after_sync();
    if (ready && !*abort) {
#pragma unroll 1
      for (int i = 0; i < kMatrices * tokens / 32; ++i) {
        const int mat = i * 32 >= tokens ? 1 : 0, c = i * 32 - mat * tokens;
        uint32_t v[32];
        tmem_load_32x32(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + mat * kMaxTokens + c, v);
        uint32_t* dst = sums + (mat * kMaxTokens + c) * kChannels + channel;
#pragma unroll
        for (int j = 0; j < 32; ++j) dst[j * kChannels] = mine > 0 ? v[j] : 0u;
      }
    }
    tc_fence_before_sync();
  }
  __syncwarp();
  cluster_sync();

  // ---- join: tokens of this part, four channels a thread ----
  const int share = (op.m + kSplit - 1) / kSplit;
  const int token0 = part * share, count = fits ? max(0, min(share, op.m - token0)) : 0;
  const uint32_t base = smem_addr(sums);
  for (int i = threadIdx.x; i < count * (kChannels / 4); i += kThreads) {
    const int token = token0 + i / (kChannels / 4), channel = 4 * (i % (kChannels / 4));
    const uint32_t at = base + (token * kChannels + channel) * 4;
    uint4 v[kSplit], u[kSplit];
#pragma unroll
    for (int p = 0; p < kSplit; ++p) {
      v[p] = read_cluster(at, p);
      if (kGated) u[p] = read_cluster(at + kMaxTokens * kChannels * 4, p);
    }
    typename T::Sum total[4] = {}, up[4] = {};
#pragma unroll
    for (int p = 0; p < kSplit; ++p) {
      add<T>(total, v[p]);
      if (kGated) add<T>(up, u[p]);
    }
    const float row_scale = T::kBlock == 128 ? op.x_scale[token] : 0.0f;
    __half* dst = op.out + static_cast<long long>(token) * op.n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int column = n0 + channel + e;
      if (column >= op.n) break;
      float y = static_cast<float>(total[e]), z = static_cast<float>(up[e]);
      if constexpr (T::kBlock == 128) {
        const float bias = !kGated && op.bias != nullptr ? __half2float(op.bias[column]) : 0.0f;
        y = ctb::dequantized(total[e], row_scale, op.w_scale[0][column], bias);
        if (kGated) z = ctb::dequantized(up[e], row_scale, op.w_scale[1][column], 0.0f);
      }
      if (kGated) y = ctb::gated(y, z, op.activation);
      dst[column] = __float2half_rn(y);
    }
  }
  if (!fits && threadIdx.x == 0) ctb::report_error(op.scratch, ctb::kErrorBadShape, 94);
  __syncwarp();
  // No CTA leaves while another one reads its sums.
  cluster_sync();
  tc_fence_after_sync();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

}  // namespace

// One argument list for all splits: those of at most 32 rows take no x64.
#define CTB_NARROW_KERNELS(split)                                                                                      \
  extern "C" __global__ void __cluster_dims__(split, 1, 1) __launch_bounds__(kThreads, 2)                              \
  ctb_gated_gemm_f16_narrow##split(const __grid_constant__ TmaDescriptor tma_x64,                                      \
                                   const __grid_constant__ TmaDescriptor tma_x32,                                      \
                                   const __grid_constant__ TmaDescriptor tma_gate,                                     \
                                   const __grid_constant__ TmaDescriptor tma_up, __half* output, int m, int n, int k,  \
                                   int activation, CTB_RESERVED_PARAMS) {                                              \
    (void)profile_scratch;                                                                                             \
    const Operands op = {&tma_x32, &tma_x64, {&tma_gate, &tma_up}, nullptr, {nullptr, nullptr}, nullptr, output,       \
                         m, n, k, activation, runtime_scratch};                                                        \
    product_narrow<Half, true, split, 32>(op);                                                                         \
  }                                                                                                                    \
  extern "C" __global__ void __cluster_dims__(split, 1, 1) __launch_bounds__(kThreads, 2)                              \
  ctb_qgemm_i8_narrow##split(const __grid_constant__ TmaDescriptor tma_x64,                                            \
                             const __grid_constant__ TmaDescriptor tma_x32,                                            \
                             const __grid_constant__ TmaDescriptor tma_w, const float* x_scale, const float* w_scale,  \
                             const __half* bias, __half* output, int m, int n, int k, CTB_RESERVED_PARAMS) {           \
    (void)profile_scratch;                                                                                             \
    const Operands op = {&tma_x32, &tma_x64, {&tma_w, nullptr}, x_scale, {w_scale, nullptr}, bias, output, m, n, k, 0, \
                         runtime_scratch};                                                                             \
    product_narrow<Int8, false, split, split >= 4 ? 64 : 32>(op);                                                      \
  }                                                                                                                    \
  extern "C" __global__ void __cluster_dims__(split, 1, 1) __launch_bounds__(kThreads, 2)                              \
  ctb_qgated_gemm_i8_narrow##split(const __grid_constant__ TmaDescriptor tma_x64,                                      \
                                   const __grid_constant__ TmaDescriptor tma_x32,                                      \
                                   const __grid_constant__ TmaDescriptor tma_gate,                                     \
                                   const __grid_constant__ TmaDescriptor tma_up, const float* x_scale,                 \
                                   const float* gate_scale, const float* up_scale, __half* output, int m, int n,       \
                                   int k, int activation, CTB_RESERVED_PARAMS) {                                       \
    (void)profile_scratch;                                                                                             \
    const Operands op = {&tma_x32, &tma_x64, {&tma_gate, &tma_up}, x_scale, {gate_scale, up_scale}, nullptr, output,   \
                         m, n, k, activation, runtime_scratch};                                                        \
    product_narrow<Int8, true, split, 32>(op);                                                                         \
  }

CTB_NARROW_KERNELS(1)
CTB_NARROW_KERNELS(2)
CTB_NARROW_KERNELS(4)
CTB_NARROW_KERNELS(8)
