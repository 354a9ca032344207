// GatedGemm, QGemm and QGatedGemm on CTA pairs (tcgen05, cta_group::2).
//
//   GatedGemm   y = act(x . Wg^T) (x . Wu^T)        FP16 operands, FP32 sums
//   QGemm       y = (q . W^T) (s[m] ws[n]) + bias   8-bit operands, 32-bit integer sums
//   QGatedGemm  both
//
// with weights [N, K] (a [K, N] constant is turned once at upload), so both
// operands are K-major rows that TMA brings in blocks of 128 bytes (64 FP16 or
// 128 8-bit k) in the 128-byte swizzle the tensor core reads; four MMAs of 32
// bytes of k each use a block up.
//
// Two CTAs of a cluster (two SMs) work on one tile of 256 rows: CTA r holds
// rows 128 r ... of x and `half` weight rows (16 to 128), and one
// tcgen05.mma.cta_group::2 (M = 256, N = 2 half) reads both halves and leaves
// 128 rows of sums in each CTA's TMEM. For the gated ops the halves are the
// same columns of the two weight matrices: CTA 0 loads gate rows, CTA 1 up
// rows, and columns c and half + c of every TMEM lane are the gate and the up
// sum of one output, so activation and product are the epilogue of the thread
// that reads them and neither projection ever leaves the SM.
//
// The width is chosen at run time (choose_half) by what a block of K costs:
// 4 half clocks of MMAs, 64 bytes a clock and SM through TMA (rows of x beyond
// M are not loaded: zero-filling them took as long as loading them), or the
// weights' share of HBM. At 512 clocks a block for half = 128 the tensor cores
// are busy throughout (8192x4096x8192: 723 us, 1520 TFLOP/s; 8 bits
// 8192x8192x4096: 171 us, 3210 TOP/s).
//
// Warp 0 loads (a ring of 192 KB), warp 1 of CTA 0 issues the MMAs into one of
// two accumulators, 16 epilogue warps of each CTA turn the other one into
// FP16 through 32 x 32 boxes that TMA stores. Tiles go round the pairs in
// blocks of kRasterRows tile rows, so that the 74 pairs at work share about
// 8 + 9 operand tiles in L2 instead of streaming all weights past each row of
// tiles. All waits are bounded (tc_common.cuh).

#include "product.cuh"
#include "tc_common.cuh"

namespace {

using namespace ctb::tc;

constexpr int kBM = 128;  // rows a CTA (the pair covers 256)
constexpr int kRowBytes = 128;
constexpr int kEpilogueWarps = 16;
constexpr int kThreads = (2 + kEpilogueWarps) * 32;
constexpr int kChunk = 32;
constexpr int kEpilogueWarp0 = 2;
constexpr int kRasterRows = 8;
constexpr uint32_t kRingBytes = 196608;
constexpr uint32_t kStageBoxBytes = 32 * kChunk * 2;
constexpr uint32_t kStagingBytes = kEpilogueWarps * kStageBoxBytes;
constexpr int kMaxStages = 10;
constexpr uint32_t kTmemCols = 512;  // two accumulators, 256 columns apart

struct Half {
  static constexpr int kBlock = 64;  // k of a 128-byte row
  // FP16 operands, FP32 sums.
  static __host__ __device__ constexpr uint32_t idesc(uint32_t m, uint32_t n) { return instr_desc(kFormatF16, m, n); }
};
struct Int8 {
  static constexpr int kBlock = 128;
  // Signed 8-bit operands (format 1), 32-bit integer sums (D format 2).
  static __host__ __device__ constexpr uint32_t idesc(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
  }
};

// Widths of a tile (weight rows a CTA) and heights of the boxes that bring
// them and the rows of x: every block of K is one copy each, since a copy costs
// its warp about 55 clocks whatever its size.
constexpr int kHalves = 5;
constexpr int kXBoxes = 3;
__device__ __forceinline__ int half_at(int i) { return i == 0 ? 128 : i == 1 ? 96 : i == 2 ? 64 : i == 3 ? 48 : 32; }
__device__ __forceinline__ int x_rows_at(int i) { return 128 >> i; }
// 64 or 32 rows a CTA where the pair's two hold all of M: a block of 128 rows
// takes 250 clocks through TMA, as long as the rest of a block's round.
__device__ __forceinline__ int x_box_for(int m) { return m > 128 ? 0 : m > 64 ? 1 : 2; }

// a / b for 0 <= a, 0 < b: the FP32 quotient is off by a few units at most
// and set right by the remainder. (An integer division by a value known at run
// time only takes some 150 clocks of a kernel's start.)
__device__ __forceinline__ int quotient(int a, int b) {
  int q = static_cast<int>(static_cast<float>(a) * ctb::reciprocal(static_cast<float>(b)));
  int r = a - q * b;
  for (; r < 0; r += b) --q;
  for (; r >= b; r -= b) ++q;
  return q;
}

// Tiles of 2^shift or 3 * 2^shift columns over n: half is 128, 64, 32 or 96, 48.
__device__ __forceinline__ int column_tiles(int n, int columns) {
  const bool three = columns % 3 == 0;  // (a compile-time divisor)
  const int shift = three ? 31 - __clz(columns / 3) : 31 - __clz(columns);
  const unsigned t = static_cast<unsigned>(n + columns - 1) >> shift;
  return static_cast<int>(three ? t / 3u : t);
}

// A tile's width and what follows from it.
struct Shape {
  int width;             // index of half
  int half;              // weight rows a CTA
  int columns;           // output columns
  int x_box;             // index of the box of x
  int rows;              // of x a CTA, the box's: the pair shares up to 64 or 128 rows out evenly
  int x_bytes, block_bytes;  // of a block of K: rows of x, and with the weight rows
  int blocks;            // of K a stage
  int stages;
  int m_tiles, n_tiles;
  int chunks;            // of 32 output columns, the last one of 16 where half is 48 and gated
  int active;            // epilogue warps a lane quarter
};

template <bool kGated>
__device__ __forceinline__ Shape shape_of(int width, int m, int n) {
  Shape s;
  s.width = width;
  s.half = half_at(width);
  s.columns = kGated ? s.half : 2 * s.half;
  s.x_box = x_box_for(m);
  s.rows = x_rows_at(s.x_box);
  s.x_bytes = s.rows * kRowBytes;
  s.block_bytes = s.x_bytes + s.half * kRowBytes;  // a multiple of 1024
  // Short blocks share a stage, one round of barriers for two or four of them
  // (128x12288x4096 in 8 bits: one 22.7, two 17.5 us; 32 rows, were they not
  // the narrow form's: one 22.1, two 17.0, four 15.0), as long as
  // enough stages are left (with three of two blocks 256x4096x12288 took 50.8
  // instead of 48.5 us).
  const int ring_blocks =
      static_cast<int>(kRingBytes * ctb::reciprocal(static_cast<float>(s.block_bytes)) + 1e-3f);  // 6 to 24
  s.blocks = ring_blocks >= 20 ? 4 : ring_blocks >= 8 ? 2 : 1;
  s.stages = min(kMaxStages, s.blocks == 4 ? ring_blocks / 4 : s.blocks == 2 ? ring_blocks / 2 : ring_blocks);
  s.m_tiles = (m + 2 * s.rows - 1) >> (8 - s.x_box);
  s.n_tiles = column_tiles(n, s.columns);
  s.chunks = (s.columns + kChunk - 1) / kChunk;
  s.active = min(s.chunks, kEpilogueWarps / 4);
  return s;
}

struct __align__(8) Barriers {
  uint64_t full[kMaxStages];   // leader: both CTAs' copies of a stage landed
  uint64_t empty[kMaxStages];  // each CTA: the stage's MMAs are done
  uint64_t tmem_full[2];       // each CTA: the accumulator is complete
  uint64_t tmem_empty[2];      // leader: the pair's epilogue warps have read it
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Without release: what the CTAs tell each other here are barrier
// initialisations (fenced by mbar_init_fence) and that they have ended; a
// releasing arrival waits for the epilogue's stores, 0.5 us and more.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t cluster_addr(const void* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(local)), "r"(rank));
  return remote;
}

// Tile load into this CTA's shared memory that counts on the leader's barrier.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const TmaDescriptor* desc, uint32_t leader_bar, int x,
                                                 int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(desc)), "r"(leader_bar), "r"(x), "r"(y)
      : "memory");
}

// Arrives on `bar` in both CTAs when this thread's earlier MMAs are done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// mbar_wait by a whole warp, which agrees on the outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, void* scratch,
                                          unsigned int site) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort, scratch, site));
}

// One lane of the warp, the same each time; the warp stays converged around it.
__device__ __forceinline__ bool elect_one() {
  uint32_t elected;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(elected));
  return elected != 0;
}

__device__ __forceinline__ void umma_pair(Half, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void umma_pair(Int8, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void arrive_on_leader(uint64_t* bar) {
  const uint32_t remote = cluster_addr(bar, 0);
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}

__device__ __forceinline__ void tma_store_2d(const TmaDescriptor* desc, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(desc)),
               "r"(smem_addr(src)), "r"(x), "r"(y)
               : "memory");
}

// Two 32 x 32 blocks of sums in one wait: 32 columns from `a` and 32 from `b`.
__device__ __forceinline__ void tmem_load_two(uint32_t a, uint32_t b, uint32_t (&v)[32], uint32_t (&u)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20,"
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50,"
      "%51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]),
        "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(a), "r"(b)
      : "memory");
}

// What the kernels bind. Scales are null in FP16.
struct Operands {
  const TmaDescriptor* x;     // the box of x that shape_of picks
  const TmaDescriptor* w[2];  // [gate / up]: the box of the tile's width
  const TmaDescriptor* out_map;
  __half* out;
  const float* x_scale;
  const float* w_scale[2];
  const __half* bias;
  int m, n, k, activation;
  void* scratch;
};

// Tile `index` in raster order: blocks of kRasterRows tile rows, within a
// block column by column.
__device__ __forceinline__ void tile_at(int index, const Shape& sh, int* mt, int* nt) {
  int first = 0;  // tile row
  if (sh.m_tiles > kRasterRows) {
    const int per_block = kRasterRows * sh.n_tiles;
    const int block = quotient(index, per_block);
    index -= block * per_block;
    first = block * kRasterRows;
  }
  const int rows = min(kRasterRows, sh.m_tiles - first);
  *nt = rows == 1 ? index : quotient(index, rows);
  *mt = first + index - *nt * rows;
}

// One lane's 32 outputs of a chunk: `v` the (gate) sums, `u` the up sums.
template <typename T, bool kGated>
__device__ __forceinline__ void finish(const Operands& op, uint32_t (&v)[kChunk], uint32_t (&u)[kChunk], int column0,
                                       float row_scale, uint4 (&packed)[kChunk / 8]) {
  constexpr bool kInt8 = T::kBlock == 128;
  const int lane = threadIdx.x & 31;
  float y[kChunk];
  if constexpr (kInt8) {
    const int column = min(column0 + lane, op.n - 1);
    // A lane is a row: it gets the columns' scales from the lanes that loaded them.
    const float c0 = op.w_scale[0][column];
    const float c1 = kGated ? op.w_scale[1][column] : 0.0f;
    const float bias = !kGated && op.bias != nullptr ? __half2float(op.bias[column]) : 0.0f;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      const float s0 = __shfl_sync(0xFFFFFFFFu, c0, j);
      const float b = kGated ? 0.0f : __shfl_sync(0xFFFFFFFFu, bias, j);
      y[j] = ctb::dequantized(static_cast<int>(v[j]), row_scale, s0, b);
      if (kGated) {
        const float s1 = __shfl_sync(0xFFFFFFFFu, c1, j);
        u[j] = __float_as_uint(ctb::dequantized(static_cast<int>(u[j]), row_scale, s1, 0.0f));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) y[j] = __uint_as_float(v[j]);
  }
  if constexpr (kGated) {
    if (op.activation == ctb::kSilu) {
#pragma unroll
      for (int j = 0; j < kChunk; ++j) y[j] = ctb::silu(y[j]) * __uint_as_float(u[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kChunk; ++j) y[j] = ctb::gelu(y[j]) * __uint_as_float(u[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < kChunk / 8; ++i) {
    __half2* h = reinterpret_cast<__half2*>(&packed[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(y[8 * i + 2 * j], y[8 * i + 2 * j + 1]);
  }
}

__device__ __forceinline__ Barriers* barriers(uint8_t* smem) {
  return reinterpret_cast<Barriers*>(smem + kRingBytes + kStagingBytes);
}

// Publishes warp 1's TMEM allocation to the issuer and the epilogue warps.
__device__ __forceinline__ uint32_t tmem_address(Barriers* bars) {
  tc_fence_before_sync();
  asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 32) : "memory");
  tc_fence_after_sync();
  return *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
}

// The MMAs of all tiles, by warp 1 of the pair's leader.
template <typename T>
__device__ __forceinline__ void issue_mmas(uint8_t* smem, Barriers* bars, const Shape& sh, uint32_t tmem, int tiles,
                                           int pair, int pairs, int k_blocks, void* scratch) {
  volatile int* abort = &bars->abort;
  const int stage_bytes = sh.blocks * sh.block_bytes;
  // The whole warp runs the loop and one lane issues, so that descriptors
  // are uniform values: by a lone thread four MMAs and two commits took 570
  // clocks a stage, more than the 512 that the tensor cores need for it.
  const uint32_t idesc = T::idesc(2 * kBM, 2 * sh.half);
  const uint64_t a_first = smem_desc_kmajor_sw128(smem);
  const uint64_t b_first = smem_desc_kmajor_sw128(smem + sh.x_bytes);
  const uint32_t empty_first = smem_addr(&bars->empty[0]);
  int s = 0;
  uint32_t phase = 0;
  bool ok = true;
  int local = 0;
  for (int tile = pair; tile < tiles && ok; tile += pairs, ++local) {
    const int buf = local & 1;
    if (local >= 2 && !warp_wait(&bars->tmem_empty[buf], ((local >> 1) - 1) & 1, abort, scratch, 72)) {
      ok = false;
      break;
    }
    tc_fence_after_sync();
    const uint32_t acc = tmem + buf * 256;
    for (int kb = 0; kb < k_blocks; kb += sh.blocks) {
      if (!warp_wait(&bars->full[s], phase, abort, scratch, 73)) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      if (elect_one()) {
        const int blocks = min(sh.blocks, k_blocks - kb);
        uint32_t offset = static_cast<uint32_t>(s * stage_bytes) >> 4;
        for (int b = 0; b < blocks; ++b, offset += static_cast<uint32_t>(sh.block_bytes) >> 4) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            umma_pair(T{}, acc, a_first + offset + 2 * kk, b_first + offset + 2 * kk, idesc, (kb | b | kk) != 0);
          }
        }
        umma_commit_pair(empty_first + 8 * s);
      }
      __syncwarp();
      if (++s == sh.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (ok && elect_one()) umma_commit_pair(smem_addr(&bars->tmem_full[buf]));
    __syncwarp();
  }
  // The peer's epilogue warps arrive here from afar: the last arrivals on both
  // accumulators have landed before this CTA may leave.
  for (int last = max(0, local - 2); ok && last < local; ++last) {
    ok = warp_wait(&bars->tmem_empty[last & 1], (last >> 1) & 1, abort, scratch, 76);
  }
  if (!ok) {
    if (elect_one()) {
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                       smem_addr(&bars->drain))
                   : "memory");
    }
    volatile int never = 0;
    mbar_wait(&bars->drain, 0, &never, scratch, 74);
    __syncwarp();
  }
}

template <typename T, bool kGated>
__device__ __forceinline__ void product_pair(uint8_t* smem, const Operands& op, const Shape sh) {
  uint8_t* staging = smem + kRingBytes;
  Barriers* bars = barriers(smem);
  volatile int* abort = &bars->abort;
  const int stage_bytes = sh.blocks * sh.block_bytes;

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pairs = gridDim.x / 2;
  const int pair = blockIdx.x / 2;
  const int k_blocks = (op.k + T::kBlock - 1) / T::kBlock;
  const int tiles = sh.m_tiles * sh.n_tiles;
  const bool tma_epilogue = op.n % 8 == 0 && ctb::aligned16(op.out);
  const TmaDescriptor* my_w = kGated && !leader ? op.w[1] : op.w[0];

  if (warp == 0) {
    // ---- TMA producer: this CTA's rows of x and of the weights ----
    const uint32_t full_first = cluster_addr(&bars->full[0], 0);  // on the leader
    int s = 0, g = 0;
    uint32_t phase = 1;  // the first round of the ring finds every stage free
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      int mt, nt;
      tile_at(tile, sh, &mt, &nt);
      const int pair_m0 = mt * 2 * sh.rows;
      const int m0 = pair_m0 + static_cast<int>(rank) * sh.rows;
      const int n0 = nt * sh.columns + (kGated ? 0 : static_cast<int>(rank) * sh.half);
      // Rows of x past M keep what the stage held: their sums are not stored,
      // and a CTA without rows loads none.
      const bool has_x = m0 < op.m;
      const int pair_bytes = 2 * sh.half * kRowBytes + (pair_m0 + sh.rows < op.m ? 2 : 1) * sh.x_bytes;
      for (int kb = 0; kb < k_blocks; kb += sh.blocks) {
        if (!warp_wait(&bars->empty[s], phase, abort, op.scratch, 70)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const int blocks = min(sh.blocks, k_blocks - kb);
          const uint32_t full = full_first + 8 * s;
          if (leader) mbar_arrive_expect_tx(&bars->full[s], blocks * pair_bytes);
          uint8_t* a = smem + s * stage_bytes;
          for (int b = 0; b < blocks; ++b, a += sh.block_bytes) {
            const int k0 = (kb + b) * T::kBlock;
            if (has_x) tma_load_2d_pair(a, op.x, full, k0, m0);
            tma_load_2d_pair(a + sh.x_bytes, my_w, full, k0, n0);
          }
        }
        __syncwarp();
        ++g;
        if (++s == sh.stages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
    // The leader's commits arrive on this CTA's stages: the last one on each has
    // landed before the CTA may leave (a stage never used passes at once).
    if (ok && lane < sh.stages) mbar_wait(&bars->empty[lane], lane < s ? phase ^ 1u : phase, abort, op.scratch, 77);
    __syncwarp();
    if (*abort && leader && lane == 0) {
      // Let the issued copies land before shared memory is released (the
      // peer's too: the leader's barrier counts them). Bounded: a phase the
      // aborted peer never fed times out after the wait limit.
      for (int q = max(0, g - sh.stages); q < g; ++q) {
        volatile int never = 0;
        mbar_wait(&bars->full[q % sh.stages], (q / sh.stages) & 1, &never, op.scratch, 71);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---- TMEM, and the MMA issuer (pair leader) ----
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars->tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    if (leader) {
      if (lane < 2) mbar_init(&bars->tmem_empty[lane], 2 * 4 * sh.active);
      mbar_init_fence();
    }
    const uint32_t tmem = tmem_address(bars);
    if (leader) issue_mmas<T>(smem, bars, sh, tmem, tiles, pair, pairs, k_blocks, op.scratch);
  } else {
    // ---- epilogue: this CTA's 128 rows, quarter = warp % 4 ----
    const uint32_t tmem = tmem_address(bars);
    const int quarter = warp & 3;
    const int wq = (warp - kEpilogueWarp0) / 4;
    uint8_t* box_smem = staging + (warp - kEpilogueWarp0) * kStageBoxBytes;
    bool box_used = false;
    // (Warps without a chunk take no part.)
    for (int tile = wq < sh.active ? pair : tiles, local = 0; tile < tiles; tile += pairs, ++local) {
      const int buf = local & 1;
      int mt, nt;
      tile_at(tile, sh, &mt, &nt);
      const int row0 = (2 * mt + static_cast<int>(rank)) * sh.rows + quarter * 32;
      const bool has_rows = quarter * 32 < sh.rows && row0 < op.m;
      const int n0 = nt * sh.columns;
      const float row_scale = op.x_scale != nullptr && has_rows && row0 + lane < op.m ? op.x_scale[row0 + lane] : 0.0f;
      const bool ready = mbar_wait(&bars->tmem_full[buf], (local >> 1) & 1, abort, op.scratch, 75);
      __syncwarp();
      if (!ready) break;
      tc_fence_after_sync();
      const uint32_t taddr = tmem + buf * 256 + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int ci = wq; ci < sh.chunks; ci += sh.active) {
        const int c = ci * kChunk;
        uint32_t v[kChunk], u[kChunk];
        if constexpr (kGated) {
          tmem_load_two(taddr + c, taddr + sh.half + c, v, u);
        } else {
          tmem_load_32x32(taddr + c, v);
        }
        if (ci + sh.active >= sh.chunks) {
          // This warp's columns are in registers: release them to the issuer.
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if (leader) {
              mbar_arrive(&bars->tmem_empty[buf]);
            } else {
              arrive_on_leader(&bars->tmem_empty[buf]);
            }
          }
        }
        // Columns past N (a partial last tile) and rows past M: nothing to store.
        if (n0 + c >= op.n || !has_rows) continue;
        uint4 packed[kChunk / 8];
        finish<T, kGated>(op, v, u, n0 + c, row_scale, packed);
        const int end = min(op.n, n0 + sh.columns);
        if (tma_epilogue && c + kChunk > sh.columns) {
          // Half a chunk (gated, half = 48): each lane its row's 32 bytes.
          if (row0 + lane < op.m) {
            __half* dst = op.out + static_cast<long long>(row0 + lane) * op.n + n0 + c;
#pragma unroll
            for (int i = 0; i < kChunk / 16; ++i) {
              if (n0 + c + 8 * i < end) *reinterpret_cast<uint4*>(dst + 8 * i) = packed[i];
            }
          }
          continue;
        }
        if (box_used) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
        }
        // Row `lane` (64 bytes); 64-byte swizzle: 16-byte chunk i at i ^ ((lane / 2) % 4).
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
          *reinterpret_cast<uint4*>(box_smem + lane * 64 + (((i ^ (lane >> 1)) & 3) << 4)) = packed[i];
        }
        if (tma_epilogue) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(op.out_map, box_smem, n0 + c, row0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          box_used = true;
        } else {
          // Rows that TMA cannot address (N no multiple of 8, an output off
          // 16 bytes): one row of the chunk a store instruction, eight under way.
          __syncwarp();
          const int column = n0 + c + lane;
          const int rows = column < end ? op.m - row0 : 0;
          __half* dst = op.out + static_cast<long long>(row0) * op.n + column;
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 8) {
            __half h[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              h[r] = *reinterpret_cast<const __half*>(
                  box_smem + (r0 + r) * 64 + ((((lane >> 3) ^ ((r0 + r) >> 1)) & 3) << 4) + (lane & 7) * 2);
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              if (r0 + r < rows) dst[static_cast<long long>(r0 + r) * op.n] = h[r];
            }
          }
          __syncwarp();
        }
      }
    }
    // The boxes have been read (the stores end with the kernel).
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  // Neither CTA leaves (or frees TMEM) while its peer may still signal it.
  cluster_arrive();
  cluster_wait();
  tc_fence_after_sync();
  if (warp == 1) {
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// The tile width with the least estimated clocks a block of K. A pair takes
// 4 half clocks of MMAs for a block plus 52, and no less than its round of
// barriers and copies (measured 295 clocks with 32 rows of x, 375 with 128).
// From HBM the weight rows of a block come at 23 bytes a clock and SM (5.6
// clocks a row) when all pairs read, shared by the m_tiles rows of tiles, and
// faster when the last wave leaves pairs idle. So few rows take the width that
// keeps HBM busy in the last wave too (64x4096x12288: half 96 or 64 44 us, 128
// 52 us, 32 49 us), many rows the widest (512x4096x11008 in 8 bits: 128 37 us,
// 64 40 us, 32 59 us), and a single wave the narrowest (100x12288x1504: 32 30
// us, 64 33 us, 128 60 us). Every warp of both CTAs gets the same answer: lane i
// rates width i, ties go to the widest.
template <bool kGated>
__device__ __forceinline__ int choose_width(int m, int n, int pairs) {
  const int lane = threadIdx.x & 31;
  const int width = min(lane, kHalves - 1);
  const float half = static_cast<float>(half_at(width));
  const int m_tiles = (m + 2 * kBM - 1) / (2 * kBM);
  const float tiles = static_cast<float>(m_tiles) * static_cast<float>(column_tiles(n, half_at(width) * (kGated ? 1 : 2)));
  const float busy = fmaxf(4.0f * half + 52.0f, 268.0f + 0.85f * static_cast<float>(x_rows_at(x_box_for(m))));
  const float hbm = 5.6f * half * ctb::reciprocal(static_cast<float>(m_tiles));
  const float waves = tiles * ctb::reciprocal(static_cast<float>(pairs));
  const float full = floorf(waves + 1e-3f);
  const float rest = fmaxf(0.0f, waves - full);
  float clocks = full * fmaxf(busy, hbm) + (rest > 1e-3f ? fmaxf(busy, hbm * rest) : 0.0f);
  if (full == 0.0f) clocks += half / 16.0f;
  const unsigned rated = static_cast<unsigned>(fminf(clocks, 2e8f)) * 8u + static_cast<unsigned>(width);
  return static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, rated) & 7u);
}

// Weight boxes of every width, by index of half.
using Boxes = const TmaDescriptor* [kHalves];

template <typename T, bool kGated>
__device__ __forceinline__ void product_dispatch(Operands& op, const TmaDescriptor* const (&x)[kXBoxes],
                                                 const Boxes& w0, const Boxes& w1) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  if (threadIdx.x < 32) {
    Barriers* bars = barriers(smem);
    const int lane = threadIdx.x;
    if (lane < 2 * kMaxStages) mbar_init(&bars->full[0] + lane, 1);  // full, then empty
    if (lane < 2) mbar_init(&bars->tmem_full[lane], 1);
    if (lane == 2) mbar_init(&bars->drain, 1);
    if (lane == 3) bars->abort = 0;
    mbar_init_fence();
  }
  // The peer's copies and commits reach these barriers: both CTAs have
  // initialised them before either goes on. The shape is computed meanwhile.
  cluster_arrive();
  const Shape sh = shape_of<kGated>(choose_width<kGated>(op.m, op.n, gridDim.x / 2), op.m, op.n);
  op.x = sh.x_box == 0 ? x[0] : sh.x_box == 1 ? x[1] : x[2];
  const auto pick = [&](const Boxes& w) {
    return sh.width == 0 ? w[0] : sh.width == 1 ? w[1] : sh.width == 2 ? w[2] : sh.width == 3 ? w[3] : w[4];
  };
  op.w[0] = pick(w0);
  op.w[1] = kGated ? pick(w1) : nullptr;
  cluster_wait();
  CTB_GRID_DEPENDENCY_SYNC();
  product_pair<T, kGated>(smem, op, sh);
}

}  // namespace

#define CTB_X_MAPS                                                                                       \
  const __grid_constant__ TmaDescriptor tma_x128, const __grid_constant__ TmaDescriptor tma_x64,         \
      const __grid_constant__ TmaDescriptor tma_x32
#define CTB_W_MAPS(name)                                                                                 \
  const __grid_constant__ TmaDescriptor name##128, const __grid_constant__ TmaDescriptor name##96,       \
      const __grid_constant__ TmaDescriptor name##64, const __grid_constant__ TmaDescriptor name##48,    \
      const __grid_constant__ TmaDescriptor name##32

extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ctb_gated_gemm_f16_pair(CTB_X_MAPS, CTB_W_MAPS(tma_gate), CTB_W_MAPS(tma_up),
                        const __grid_constant__ TmaDescriptor tma_out, __half* output, int m, int n, int k,
                        int activation, CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  Operands op = {nullptr, {nullptr, nullptr}, &tma_out, output, nullptr, {nullptr, nullptr}, nullptr, m, n, k,
                 activation, runtime_scratch};
  product_dispatch<Half, true>(op, {&tma_x128, &tma_x64, &tma_x32},
                               {&tma_gate128, &tma_gate96, &tma_gate64, &tma_gate48, &tma_gate32},
                               {&tma_up128, &tma_up96, &tma_up64, &tma_up48, &tma_up32});
}

extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ctb_qgemm_i8_pair(CTB_X_MAPS, CTB_W_MAPS(tma_w), const __grid_constant__ TmaDescriptor tma_out, const float* x_scale,
                  const float* w_scale, const __half* bias, __half* output, int m, int n, int k,
                  CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  Operands op = {nullptr, {nullptr, nullptr}, &tma_out, output, x_scale, {w_scale, nullptr}, bias, m, n, k, 0,
                 runtime_scratch};
  product_dispatch<Int8, false>(op, {&tma_x128, &tma_x64, &tma_x32},
                                {&tma_w128, &tma_w96, &tma_w64, &tma_w48, &tma_w32},
                                {&tma_w128, &tma_w96, &tma_w64, &tma_w48, &tma_w32});
}

extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
ctb_qgated_gemm_i8_pair(CTB_X_MAPS, CTB_W_MAPS(tma_gate), CTB_W_MAPS(tma_up),
                        const __grid_constant__ TmaDescriptor tma_out, const float* x_scale, const float* gate_scale,
                        const float* up_scale, __half* output, int m, int n, int k, int activation,
                        CTB_RESERVED_PARAMS) {
  (void)profile_scratch;
  Operands op = {nullptr, {nullptr, nullptr}, &tma_out, output, x_scale, {gate_scale, up_scale}, nullptr, m, n, k,
                 activation, runtime_scratch};
  product_dispatch<Int8, true>(op, {&tma_x128, &tma_x64, &tma_x32},
                               {&tma_gate128, &tma_gate96, &tma_gate64, &tma_gate48, &tma_gate32},
                               {&tma_up128, &tma_up96, &tma_up64, &tma_up48, &tma_up32});
}
