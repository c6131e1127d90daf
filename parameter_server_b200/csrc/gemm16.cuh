// Matrix products of 16-bit operands on the tensor cores with an epilogue of the caller's: D[M,N] = A[M,K] · B[N,K]ᵀ,
// fp32 accumulation in TMEM, one launch for a batch of them.
//
// Operands.  An operand is one 16-bit matrix or, where fp32 accuracy is wanted, two planes of fp16: x·2^s = hi + lo with
// hi = fp16(x·2^s) and lo = fp16(x·2^s − hi), which together carry 22 bits.  The product is then the sum of hi·hi, hi·lo
// and lo·hi in one accumulator; what is left out, lo·lo, is below 2^-22 of the terms.  That costs three 16-bit products
// where three tf32 products (11 bits as well) would cost six.  The tensor cores cut a sum to fp32 at every step of 16
// elements instead of rounding it, an error that grows with the number of steps (K = 60,000: 6e-5 of a gradient); products
// of planes are therefore summed in TMEM for 128 elements of K at a time (24 steps) and added up in the epilogue's
// registers.  (64 elements: 25 % slower; 256: 4 % faster, twice the error.)  Products of 16-bit operands are summed in
// TMEM for as many elements at a time as the epilogue says (kLongK): 32,768 where results are of 16 bits (a sum of one sign comes out
// 2^-14 short; 6,000,000 elements in one sum: 1 %), 4096 for scores, which are fp32 (2^-17).  An operand may lie either way round in memory: K-major
// ([rows][k], k contiguous) or MN-major ([k][rows], rows contiguous); nothing is transposed in memory.
//
// Shape.  Persistent CTAs, or CTA pairs (cta_group::2) where the problem has enough tiles:
//   warp 0, one lane    TMA producer, a ring of stages of 64 elements of K (128-byte swizzle rows)
//   warp 1, one lane    tcgen05.mma; in a pair the leader issues for both CTAs
//   warps 4-11 or -19   epilogue: warp w reads TMEM lanes 32(w % 4)..+31, half or a quarter of the tile's columns; TMEM holds
//                       two or more accumulators, so a tile's epilogue runs under the next tile's products
// Sums of planes need 128 registers of an epilogue thread: its warps take over registers of the other four.
// 16-bit results leave through shared memory as TMA stores of 32 x 32 boxes: a lane holds a row, and stores of rows by
// lanes touch 32 lines an instruction (4096 x 4096 Newton-Schulz step: 2.6 times the time; 16-byte stores of what the warp
// turned round in shared memory: 1.05 times).
// Launches of one call overlap: a kernel sets itself up while the one before it drains (programmatic dependent launch) and
// waits for it before it touches memory.
// No load is a multicast.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "psb_tcgen05.cuh"

namespace psb {

constexpr int kG16K = 64;
constexpr int kG16Epi = 4;                         // first warp of the epilogue
constexpr int kG16Smem = 225 * 1024;              // of the stages and of what leaves
constexpr int kBoxBytes = 2048;                   // 32 x 32 values of 16 bits


// kLong: blocks of K that 16-bit operands are summed over in TMEM, 0: all
template <int kCtas_, int kN_, int kPlanes_, int kParts_ = 2, int kLong = 0>
struct Cfg16 {
  static constexpr int kCtas = kCtas_, kN = kN_, kPlanes = kPlanes_;
  static constexpr int kM = 128 * kCtas, kBRows = kN / kCtas;
  static constexpr int kABytes = 128 * 128, kBBytes = kBRows * 128;
  static constexpr int kStageBytes = kPlanes * (kABytes + kBBytes);
  // Epilogue warps for each 32 lanes of TMEM, and 4 KB of shared memory for the stores of each
  static constexpr int kParts = kParts_, kPart = kN / kParts;
  static constexpr int kThreads = 128 + 128 * kParts, kBoxes = 2;
  static constexpr int kFit = (kG16Smem - 4 * kParts * kBoxes * kBoxBytes) / kStageBytes, kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kSmemBytes = kStages * kStageBytes + 4 * kParts * kBoxes * kBoxBytes + 1024 + 512;
  static constexpr int kBufs = 512 / kN;           // accumulators in TMEM: products run ahead of the epilogue by so many less one
  static constexpr bool kPromote = kPlanes == 2 || kLong > 0;   // sums of kChunk blocks of K are added up in registers
  static constexpr int kChunk = kPlanes == 2 ? 2 : kLong > 0 ? kLong : 1 << 30;
  static_assert(kStages >= 3 && kBRows % 64 == 0 && kBufs >= 2 && kSmemBytes <= 232448, "shape of a tile");
};

struct Gemm16Args {
  CUtensorMap a, b;
  int M, N, K, batch;
  int a_z, b_z;                // matrices of a map per batch entry (planes that lie there, whether read or not); 0: one for all
  int a_m0, a_k0, b_n0, b_k0;  // where the problem starts in the maps
  int splits, kb_split;        // K blocks are dealt to `splits` pieces of kb_split; a piece is a tile of its own
  int a_mn, b_mn;              // an operand is MN-major
  int sym;                     // square result that is symmetric: only tiles on and above the diagonal
  int bf16;                    // operands are bf16, else fp16
  int a_bytes, b_bytes;        // of a stage and plane that copies bring (launch16 sets them and k_steps)
  int k_steps;                 // steps of 16 elements in a block of K
  uint32_t* status;
};

// One product, or two whose tiles are dealt to the CTAs as one list: small ones that do not depend on one another.  (How many
// is known to the compiler: arguments at an address that is not cost a large product 3 %.)
template <class Epi, int kCount>
struct Launch16 {
  Gemm16Args g[kCount];
  typename Epi::Params ep[kCount];
};

struct Tile16 {
  int z, split, m0, n0, kb0, kb1, tn;
  bool mirror;                 // the tile lies above the diagonal of a symmetric result
};

template <class C>
__host__ __device__ __forceinline__ int tiles16(const Gemm16Args& g) {
  const int tm = (g.M + C::kM - 1) / C::kM, tn = (g.N + C::kN - 1) / C::kN;
  return g.batch * g.splits * (g.sym ? tm * (tm + 1) / 2 : tm * tn);
}

// A CTA's (or pair's) tiles, every step-th from the first on.  The dimension with fewer tiles runs fastest: its operand stays in
// L2 while the other one is read once.  Counted up digit by digit: the divisions that find a tile by its number are a fifth
// of the time that the epilogue of a tile of short K has.
template <class C>
struct Tiles16 {
  const Gemm16Args& g;
  int tm, tn, nf, ns, fast, slow, zs, by_fast, by_slow, by_zs;
  __device__ __forceinline__ Tiles16(const Gemm16Args& g_, int first, int step) : g(g_) {
    tm = (g.M + C::kM - 1) / C::kM;
    tn = (g.N + C::kN - 1) / C::kN;
    nf = g.sym ? tm * (tm + 1) / 2 : tm <= tn ? tm : tn;
    ns = g.sym ? 1 : tm <= tn ? tn : tm;
    fast = first % nf; by_fast = step % nf;
    first /= nf; step /= nf;
    slow = first % ns; by_slow = step % ns;
    zs = first / ns; by_zs = step / ns;
  }
  __device__ __forceinline__ bool more() const { return zs < g.batch * g.splits; }
  __device__ __forceinline__ void next() {
    fast += by_fast; slow += by_slow; zs += by_zs;
    if (fast >= nf) { fast -= nf; ++slow; }
    if (slow >= ns) { slow -= ns; ++zs; }
  }
  __device__ __forceinline__ Tile16 get() const {
    Tile16 w;
    w.z = g.splits == 1 ? zs : zs / g.splits;
    w.split = g.splits == 1 ? 0 : zs - w.z * g.splits;
    int i = tm <= tn ? fast : slow, j = tm <= tn ? slow : fast;
    if (g.sym) {                           // the fast-th tile on and above the diagonal, column by column
      j = (int)((sqrtf(8.f * (float)fast + 1.f) - 1.f) * 0.5f);
      while ((j + 1) * (j + 2) / 2 <= fast) ++j;
      while (j * (j + 1) / 2 > fast) --j;
      i = fast - j * (j + 1) / 2;
    }
    w.mirror = g.sym && i != j;
    w.m0 = i * C::kM; w.n0 = j * C::kN; w.tn = j;
    const int nkb = (g.K + kG16K - 1) / kG16K;
    w.kb0 = w.split * g.kb_split;
    w.kb1 = w.kb0 + g.kb_split < nkb ? w.kb0 + g.kb_split : nkb;
    return w;
  }
};

template <int kCtas>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (kCtas == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// rows r0.. of an operand, K block k0, into `rows` swizzled rows of 128 bytes (K-major) or into chunks of 64 rows, each
// 64 k-lines of 128 bytes (MN-major)
template <int kCtas, int kRows>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, uint32_t bar, int k0, int r0, int z, bool mn) {
  if (mn) {
#pragma unroll
    for (int c = 0; c < kRows / 64; ++c) tma_load_3d<kCtas>(dst + c * 8192, map, bar, r0 + c * 64, k0, z);
  } else {
    tma_load_3d<kCtas>(dst, map, bar, k0, r0, z);
  }
}
// MN-major, 128-byte swizzle: a chunk of 64 rows is 64 k-lines of 128 bytes, 8 lines are a swizzle atom.  Leading
// byte offset (bits 16-29): from a chunk to the next, 8192; stride byte offset: from 8 k-lines to the next, 1024.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn) {
  return make_smem_desc(addr) | (mn ? (uint64_t)(8192 >> 4) << 16 : 0ull);
}
// kind::f16: D fp32, A and B fp16 (0) or bf16 (1) at bits 7-9 and 10-12, bits 15 / 16: A / B is MN-major
template <class C>
__device__ __forceinline__ uint32_t idesc16(const Gemm16Args& g) {
  return (1u << 4) | ((uint32_t)g.bf16 << 7) | ((uint32_t)g.bf16 << 10) | ((uint32_t)(g.a_mn != 0) << 15) | ((uint32_t)(g.b_mn != 0) << 16)
         | ((uint32_t)(C::kN >> 3) << 17) | ((uint32_t)(C::kM >> 4) << 24);
}
template <int kCtas>
__device__ __forceinline__ void mma16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kCtas == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <int kCtas>
__device__ __forceinline__ void commit16(uint64_t* bar) {
  if constexpr (kCtas == 2) commit_pair(bar);
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Wait until the launches before this one are complete and their writes visible, then let the next one start its set-up.  What a
// launch before wrote is read through pointers without __restrict__: the kernel may be running while it is written, so that it
// is no read-only data, whose loads may be moved before the wait.
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// hi and lo plane of a value that is scaled already
__device__ __forceinline__ void split16(float v, __half& hi, __half& lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}
__device__ __forceinline__ uint32_t pack_half2(__half a, __half b) {
  return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16);
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// the columns from col to col + kPart of a row of n floats, towards L2
template <int kPart>
__device__ __forceinline__ void prefetch_l2(const float* row, int col, int n) {
#pragma unroll
  for (int c = 0; c < kPart; c += 32)
    if (col + c < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + col + c));
}

enum : int { kFmtF16 = 0, kFmtBF16 = 1, kFmtPlanes = 2 };      // fp16, bf16, hi and lo planes of fp16

// two neighbouring values in the format's halves, or what the high plane leaves of them
template <int fmt>
__device__ __forceinline__ uint32_t pair16(float x, float y, bool low) {
  if constexpr (fmt == kFmtBF16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(x, y);
    if (fmt == kFmtPlanes && low) {
      const float2 b = __half22float2(t);
      t = __floats2half2_rn(x - b.x, y - b.y);
    }
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}
// An epilogue warp's way to global memory: its shared memory, kBoxes boxes.  v: 32 columns from col on of this lane's row of the
// 32 rows from row on.
template <int kBoxes>
struct OutStage {
  uint32_t addr;
  float* f;
  int lane;

  uint32_t turn = 0;

  // The buffer that the next store uses, free again: a store takes some 1000 cycles until its box has been read.
  __device__ __forceinline__ uint32_t acquire() {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kBoxes - 1) : "memory");
    __syncwarp();
    return addr + (turn++ % kBoxes) * (uint32_t)kBoxBytes;
  }
  // 32 x 32 boxes in the format, a plane at a time, as they are and, for a mirror image, transposed.  Rows of 64 bytes, 64-byte
  // swizzle (16-byte piece j of row r lies at j ^ ((r / 2) % 4)): free of bank conflicts.  What lies outside the map is not
  // written.  A tile's epilogue runs once or a few times a launch, so its code is kept short.
  template <int fmt>
  __device__ __forceinline__ void store(const CUtensorMap* map, const float (&v)[32], int row, int col, int z, bool mirror) {
    const int planes = fmt == kFmtPlanes ? 2 : 1, passes = mirror ? 2 * planes : planes;
#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {
      const bool turned = pass >= planes, low = fmt == kFmtPlanes && (pass & 1);
      uint32_t h[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) h[j] = pair16<fmt>(v[2 * j], v[2 * j + 1], low);
      const uint32_t a = acquire();
      if (!turned) {
        const uint32_t mine = a + (uint32_t)lane * 64u, sw = ((uint32_t)lane >> 1) & 3u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + (((uint32_t)j ^ sw) << 4)), "r"(h[4 * j]), "r"(h[4 * j + 1]),
                       "r"(h[4 * j + 2]), "r"(h[4 * j + 3]) : "memory");
      } else {                                             // row j holds column j, this lane's element
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t at = a + (uint32_t)j * 128u + ((((uint32_t)lane >> 3) ^ ((uint32_t)j & 3u)) << 4) + ((uint32_t)lane & 7u) * 2u;
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"((uint16_t)h[j]) : "memory");
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + 64u), "h"((uint16_t)(h[j] >> 16)) : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                     ::"l"(map), "r"(turned ? row : col), "r"(turned ? col : row), "r"(z + low), "r"(a) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
  }
  __device__ __forceinline__ void drain() {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  // Results of any stride and alignment: f(r, v) for r = 0..31 with v = row r's value of column `lane`, so that a warp's
  // accesses are pieces of one row.  The exclusive or keeps both directions free of bank conflicts.  Boxes of the tile before, which
  // may be another product's of the launch and go by store(), have been read before they are overwritten.
  template <class F>
  __device__ __forceinline__ void by_rows(const float (&v)[32], F f) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 32; ++j) f32(lane, j) = v[j];
    __syncwarp();
    f([&](int r) { return f32(r, lane); });
  }
  __device__ __forceinline__ float& f32(int r, int c) { return f[r * 32 + (c ^ r)]; }
};

// 32 sums of the warp's part of a tile from column c on: from TMEM, or from the registers that they were added up in
template <int kPart>
struct SumsInTmem {
  uint32_t taddr;
  __device__ __forceinline__ void load(int c, float (&v)[32]) const {
    uint32_t r[32];
    __syncwarp();                        // lanes may have gone apart over the columns before; the load is the whole warp's
    tmem_load_32x32(taddr + (uint32_t)c, r);
    tmem_load_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
  }
};
template <int kPart>
struct SumsInRegisters {
  const float (&sum)[kPart];
  __device__ __forceinline__ void load(int c, float (&v)[32]) const {       // by selection, so that loops over c need not be unrolled
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      float t = sum[j];
#pragma unroll
      for (int k = 32; k < kPart; k += 32) t = c == k ? sum[k + j] : t;
      v[j] = t;
    }
  }
};

// An epilogue is a struct with Params and
//   run<kPlanes, kPart>(params, args, tile, row, col, part, stage, sums, done)
// row: the first of the warp's 32 rows, col: the first of its kPart columns, the tile's part-th (either may lie outside the result); done() is
// called after the last load of sums.  ahead<kPart>(params, tile, row, col, lane) is called while the products of the tile are
// made, for what the epilogue is going to read.
template <class C, class Epi, int kCount>
__global__ void __launch_bounds__(C::kThreads, 1)
gemm16_kernel(const __grid_constant__ Launch16<Epi, kCount> launch) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* outs = stages + C::kStages * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(outs + 4 * C::kParts * C::kBoxes * kBoxBytes);
  uint64_t *empty = full + C::kStages, *tfull = empty + C::kStages, *tempty = tfull + C::kBufs;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(tempty + C::kBufs);
  volatile uint32_t* abort_flag = tmem_base + 1;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = C::kCtas == 2 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / C::kCtas, step = gridDim.x / C::kCtas;
  // the second product's tiles follow the first's
  const int first1 = kCount > 1 ? (first + step - tiles16<C>(launch.g[0]) % step) % step : 0;

  if (threadIdx.x == 32) {
    for (int pr = 0; pr < kCount; ++pr) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&launch.g[pr].a) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&launch.g[pr].b) : "memory");
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < C::kBufs; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], 4 * C::kParts * C::kCtas); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    if constexpr (C::kCtas == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (C::kCtas == 2) cluster_sync_all();       // the peer's barriers are ready before anything is signalled there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_base, 0);
  pdl_wait();

  if (warp < kG16Epi) {
    if constexpr (C::kPromote) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");    // 384 x 168 registers at launch = 128 x 56 + 256 x 224
    bool ok = true;                       // the same in all lanes of a warp
    if (warp == 0) {
      uint32_t it = 0;
      for (int pr = 0; pr < kCount; ++pr) {
        const Gemm16Args& g = launch.g[pr];
        for (Tiles16<C> t(g, pr == 0 ? first : first1, step); t.more() && ok; t.next()) {
          const Tile16 w = t.get();
          const int am = g.a_m0 + w.m0 + rank * 128, bn = g.b_n0 + w.n0 + rank * C::kBRows;
          for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
            const int st = it % C::kStages;
            if (it >= (uint32_t)C::kStages && !(ok = mbar_wait_warp(&empty[st], ((it / C::kStages) - 1) & 1))) break;
            const uint32_t bar = C::kCtas == 2 ? mapa_u32(smem_u32(&full[st]), 0) : smem_u32(&full[st]);
            const uint32_t sa = smem_u32(stages) + st * C::kStageBytes, sb = sa + C::kPlanes * C::kABytes;
            if (elect_one()) {
              if (rank == 0) mbar_expect_tx(&full[st], (uint32_t)(C::kCtas * C::kPlanes * (g.a_bytes + g.b_bytes)));
#pragma unroll
              for (int p = 0; p < C::kPlanes; ++p) {
                load_operand<C::kCtas, 128>(sa + p * C::kABytes, &g.a, bar, g.a_k0 + kb * kG16K, am, w.z * g.a_z + p, g.a_mn);
                load_operand<C::kCtas, C::kBRows>(sb + p * C::kBBytes, &g.b, bar, g.b_k0 + kb * kG16K, bn, w.z * g.b_z + p, g.b_mn);
              }
            }
            __syncwarp();
          }
          ok = ok && __all_sync(0xffffffffu, *abort_flag == 0);
        }
      }
      // the last releases must have landed here before this CTA's shared memory may go away
      for (uint32_t u = it > (uint32_t)C::kStages ? it - C::kStages : 0; u < it && ok; ++u) ok = mbar_wait_warp(&empty[u % C::kStages], (u / C::kStages) & 1);
      if (!ok) *abort_flag = 1;
    } else if (warp == 1 && rank == 0) {
      uint32_t it = 0, n = 0;
      for (int pr = 0; pr < kCount; ++pr) {
        const Gemm16Args& g = launch.g[pr];
        const uint32_t idesc = idesc16<C>(g);
        // 16 elements of K: 32 bytes of a K-major row, 16 lines of 128 bytes MN-major
        const uint64_t ka = g.a_mn ? 2048 >> 4 : 32 >> 4, kb_ = g.b_mn ? 2048 >> 4 : 32 >> 4;
        const uint64_t base_a = operand_desc(smem_u32(stages), g.a_mn), base_b = operand_desc(smem_u32(stages) + C::kPlanes * C::kABytes, g.b_mn);
        for (Tiles16<C> t(g, pr == 0 ? first : first1, step); t.more() && ok; t.next()) {
          const Tile16 w = t.get();
          for (int kc = w.kb0; kc < w.kb1 && ok; kc += C::kChunk, ++n) {
            const uint32_t acc = n % C::kBufs;
            if (n >= C::kBufs && !(ok = mbar_wait_warp(&tempty[acc], (n / C::kBufs - 1) & 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + acc * (uint32_t)C::kN;
            const int ke = w.kb1 - kc < C::kChunk ? w.kb1 : kc + C::kChunk;
            uint32_t accumulate = 0;
            for (int kb = kc; kb < ke; ++kb, ++it) {
              const int st = it % C::kStages;
              if (!(ok = mbar_wait_warp(&full[st], (it / C::kStages) & 1))) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              const uint64_t sa = base_a + (uint32_t)(st * (C::kStageBytes >> 4)), sb = base_b + (uint32_t)(st * (C::kStageBytes >> 4));
              if (elect_one()) {
#pragma unroll
                for (int q = 0; q < (C::kPlanes == 2 ? 3 : 1); ++q) {      // hi·lo, lo·hi, hi·hi
                  const uint64_t da = sa + (q == 1 ? C::kABytes >> 4 : 0), db = sb + (C::kPlanes == 2 && q == 0 ? C::kBBytes >> 4 : 0);
#pragma unroll
                  for (int k = 0; k < kG16K / 16; ++k)
                    if (k < g.k_steps) mma16<C::kCtas>(d, da + k * ka, db + k * kb_, idesc, q == 0 && k == 0 ? accumulate : 1u);
                }
                commit16<C::kCtas>(&empty[st]);
              }
              __syncwarp();
              accumulate = 1;
            }
            if (ok && elect_one()) commit16<C::kCtas>(&tfull[acc]);
            __syncwarp();
          }
          ok = ok && __all_sync(0xffffffffu, *abort_flag == 0);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    if constexpr (C::kPromote) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    constexpr int kPart = C::kPart;
    const int q = warp & 3, part = (warp - kG16Epi) >> 2;
    uint8_t* mine = outs + (warp - kG16Epi) * (C::kBoxes * kBoxBytes);
    OutStage<C::kBoxes> stage{smem_u32(mine), reinterpret_cast<float*>(mine), lane};
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(part * kPart);
    uint32_t n = 0;
    // warp-uniform, as the TMEM loads are warp-collective
    auto sums_ready = [&](uint32_t acc, uint32_t parity) {
      int ok = 1;
      if (lane == 0) {
        ok = mbar_wait(&tfull[acc], parity) ? 1 : 0;
        if (!ok) *abort_flag = 1;
        if (*abort_flag) ok = 0;
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return ok != 0;
    };
    auto release = [&](uint32_t acc) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if constexpr (C::kCtas == 2)
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapa_u32(smem_u32(&tempty[acc]), 0)) : "memory");
        else
          asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&tempty[acc])) : "memory");
      }
    };
    bool ok = true;
    for (int pr = 0; pr < kCount; ++pr) {
      const Gemm16Args& g = launch.g[pr];
      const typename Epi::Params& ep = launch.ep[pr];
      for (Tiles16<C> t(g, pr == 0 ? first : first1, step); t.more() && ok; t.next()) {
        const Tile16 w = t.get();
        const int row = w.m0 + rank * 128 + q * 32, col = w.n0 + part * kPart;
        Epi::template ahead<kPart>(ep, w, row, col, lane);
        if constexpr (C::kPromote) {
          float sum[kPart];
#pragma unroll
          for (int j = 0; j < kPart; ++j) sum[j] = 0.f;
          for (int kc = w.kb0; kc < w.kb1; kc += C::kChunk, ++n) {
            const uint32_t acc = n % C::kBufs;
            if (!(ok = sums_ready(acc, (n / C::kBufs) & 1))) break;
            uint32_t r[2][32];
            __syncwarp();
            tmem_load_32x32(lanes + acc * (uint32_t)C::kN, r[0]);
#pragma unroll
            for (int c = 0; c < kPart; c += 32) {      // the next load is on its way while these are added
              tmem_load_wait();
              if (c + 32 < kPart) tmem_load_32x32(lanes + acc * (uint32_t)C::kN + (uint32_t)c + 32u, r[(c / 32 + 1) & 1]);
              else release(acc);
#pragma unroll
              for (int j = 0; j < 32; ++j) sum[c + j] += __uint_as_float(r[(c / 32) & 1][j]);
            }
          }
          if (!ok) break;
          Epi::template run<C::kPlanes, kPart>(ep, g, w, row, col, part, stage, SumsInRegisters<kPart>{sum}, [] {});
        } else {
          const uint32_t acc = n % C::kBufs;
          if (!(ok = sums_ready(acc, (n / C::kBufs) & 1))) break;
          ++n;
          Epi::template run<C::kPlanes, kPart>(ep, g, w, row, col, part, stage, SumsInTmem<kPart>{lanes + acc * (uint32_t)C::kN}, [&] { release(acc); });
        }
      }
    }
    stage.drain();
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) set_status(launch.g[0].status, kWaitTimeout, blockIdx.x, 400);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (C::kCtas == 2) cluster_sync_all();       // neither CTA frees its accumulators or leaves while the other still works
  if (warp == 0) {
    if constexpr (C::kCtas == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

}  // namespace psb

namespace {

constexpr int kMaxDevices = 64;

int sm_count(int* dev_out) {
  static int sms[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  *dev_out = dev;
  return sms[dev];
}

// Map over `count` row-major 16-bit matrices of [rows][cols], row stride ld elements, matrix stride `stride` elements;
// the box is 64 columns of box_rows rows, 32 of 32 for results (out).  0, a driver error, or -1 without the driver's entry point.
int make_map16(CUtensorMap* map, const void* base, int bf16, int64_t rows, int64_t cols, int64_t ld, int64_t stride, int count, int box_rows,
               bool out = false) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return -1;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(count > 1 ? stride : ld * rows) * 2};
  const cuuint32_t box[3] = {out ? 32u : 64u, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
  return (int)enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box,
                  estr, CU_TENSOR_MAP_INTERLEAVE_NONE, out ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// One 16-bit matrix, or `planes` of them `plane_stride` elements apart per batch entry, as a caller describes it
struct Operand16 {
  const void* base;
  int64_t rows, cols, ld, stride;     // of the memory: rows of `cols` contiguous elements
  int count;                          // matrices in the map
};

int make_out_map(CUtensorMap* map, const Operand16& o, int bf16) {
  return make_map16(map, o.base, bf16, o.rows, o.cols, o.ld, o.stride, o.count, 32, true);
}

// A launch of a call: every one after the first may start its set-up before its predecessor is complete.
struct Chain {
  cudaStream_t stream;
  bool started = false;
  template <class... P, class... A>
  int launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, int cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (cluster > 1) {
      at[n].id = cudaLaunchAttributeClusterDimension;
      at[n].val.clusterDim.x = (unsigned)cluster; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
      ++n;
    }
    if (started) {
      at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[n].val.programmaticStreamSerializationAllowed = 1;
      ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = (unsigned)n;
    started = true;
    return (int)cudaLaunchKernelEx(&cfg, kernel, (P)args...);
  }
};

// what the device needs to know of a product's operands
template <class C>
int set_operands(psb::Gemm16Args& g, const Operand16& a, const Operand16& b) {
  // A copy that fills in rows from outside a matrix takes 2 to 3 cycles a row: one row of x in a box of 128 made scores of
  // 400,000 classes take 190 us instead of 134.  Boxes are no higher than the matrix.  Rows of K-major operands that no copy
  // brings may hold anything: their results are rows or columns that do not exist.  Lines of MN-major operands are
  // elements of K: all of those that a step of 16 multiplies are brought, zeros behind the last.
  auto up = [](int64_t v, int by, int most) { return v >= most ? most : (int)((v + by - 1) / by * by); };
  const int lines = up(g.K, 16, psb::kG16K), ra = g.a_mn ? lines : up(g.M, 8, 128), rb = g.b_mn ? lines : up(g.N, 8, C::kBRows);
  int r = make_map16(&g.a, a.base, g.bf16, a.rows, a.cols, a.ld, a.stride, a.count, ra);
  if (r == 0) r = make_map16(&g.b, b.base, g.bf16, b.rows, b.cols, b.ld, b.stride, b.count, rb);
  if (r) return r;
  g.a_bytes = ra * 128 * (g.a_mn ? 2 : 1);
  g.b_bytes = rb * 128 * (g.b_mn ? C::kBRows / 64 : 1);
  g.k_steps = lines / 16;
  return 0;
}

template <class C, class Epi, int kCount>
int launch16(Chain& chain, psb::Launch16<Epi, kCount>& launch, const Operand16* a, const Operand16* b) {
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms <= 0) return (int)cudaErrorInvalidDevice;
  int tiles = 0;
  for (int pr = 0; pr < kCount; ++pr) {
    const int r = set_operands<C>(launch.g[pr], a[pr], b[pr]);
    if (r) return r;
    tiles += psb::tiles16<C>(launch.g[pr]);
  }
  static bool attr[kMaxDevices] = {};
  if (!attr[dev]) {
    cudaError_t e = cudaFuncSetAttribute(psb::gemm16_kernel<C, Epi, kCount>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    cudaFuncAttributes fa;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, psb::gemm16_kernel<C, Epi, kCount>);
    if (e != cudaSuccess) return (int)e;
    // the epilogue's warps wait for registers that the launch has to have brought
    if (C::kPromote && fa.numRegs * C::kThreads < 128 * 56 + 256 * 224) return (int)cudaErrorLaunchOutOfResources;
    attr[dev] = true;
  }
  const int most = sms / C::kCtas;
  return chain.launch(psb::gemm16_kernel<C, Epi, kCount>, dim3((unsigned)((tiles < most ? tiles : most) * C::kCtas)), C::kThreads, C::kSmemBytes, C::kCtas, launch);
}

// ---- which tiles, and in how many pieces K is taken
// 256x256 on a pair, with two or four epilogue warps for 32 rows, 256x128 on a pair, 128x128, 128x64
enum : int { kPair256 = 0, kPair128 = 1, kOne128 = 2, kOne64 = 3, kKinds = 4, kPair256Wide = 4 };
struct Tiling { int kind, splits, kb_split, sym; };

inline int tiling_rows(int kind) { return kind <= kPair128 || kind == kPair256Wide ? 256 : 128; }
inline int tiling_cols(int kind) { return kind == kPair256 || kind == kPair256Wide ? 256 : kind == kOne64 ? 64 : 128; }
inline int tiling_parts(int kind) { return kind == kPair256Wide ? 4 : 2; }

// The cheapest by this estimate, in cycles of an SM.  A round of tiles costs its blocks of K, at the slower of the tensor
// cores (128 x N x 64 in 2N cycles a product) and the loads (48 bytes a cycle), or the epilogue where that takes longer:
// 700 cycles for 32 rows x 32 columns of a plane and a warp, by clock readings (`outputs` of them, twice for a mirror image).
// The last round's epilogue comes on top; with two planes, whose sums are in its warps' registers, that of every round.  Pieces of
// K cost a launch that adds them up and their bytes, 5000 a cycle.  A symmetric product may make all tiles: where one round
// holds them, that saves the mirror images (512 x 512, two planes: 22 -> 14 k cycles).
inline Tiling choose_tiling(int64_t batch, int64_t M, int64_t N, int64_t K, int planes, bool symmetric, int max_splits, int outputs = 1,
                            int only = -1) {
  const int64_t nkb = (K + psb::kG16K - 1) / psb::kG16K;
  Tiling best = {kOne64, 1, (int)nkb, 0};
  double least = 1e300;
  for (int kind = 0; kind < kKinds; ++kind) {
    if (only >= 0 && kind != only) continue;
    const int64_t rows = tiling_rows(kind), cols = tiling_cols(kind);
    const int64_t tm = (M + rows - 1) / rows, tn = (N + cols - 1) / cols, slots = rows == 256 ? 74 : 148;
    for (int sym = 0; sym <= (symmetric && rows == cols ? 1 : 0); ++sym) {
      const int64_t tiles = batch * (sym ? tm * (tm + 1) / 2 : tm * tn);
      const double mma = 2.0 * cols * (planes == 2 ? 3 : 1);
      const double load = planes * (16384.0 + 128.0 * cols * 128.0 / rows) / 48.0;
      const double plain = 700.0 * cols / 64.0, epilogue = plain * planes * outputs * (sym && tm > 1 ? 1.8 : 1.0);
      for (int64_t s = 1; s <= max_splits && s <= nkb; ++s) {
        const int64_t per = (nkb + s - 1) / s, real = (nkb + per - 1) / per;
        if (real != s) continue;
        if (s > 1 && per < 4) break;
        const double rounds = (double)((tiles * s + slots - 1) / slots), main = (double)per * (mma > load ? mma : load);
        const double e = s > 1 ? 2.0 * plain : epilogue;          // fp32 sums of a piece
        double t = planes == 2 ? rounds * (main + e + 600.0) : rounds * ((main > e ? main : e) + 600.0) + e;
        if (s > 1) t += 5000.0 + (double)batch * M * N * (8.0 * s + 4.0) / 5000.0;
        if (t < least) { least = t; best = {kind, (int)s, (int)per, sym}; }
      }
    }
  }
  // One plane: up to K = 768 a tile's products take less time than its epilogue, where two warps wait out each other's loads
  // and exponentials (4096 x 65,536 scores, K = 512: 296 -> 208 us; K = 1024, 2 % slower: a stage less, more power).
  if (best.kind == kPair256 && planes == 1 && best.kb_split <= 12) best.kind = kPair256Wide;
  return best;
}

template <int kPlanes, int kLong, class Epi>
int launch_kind(Chain& chain, int kind, psb::Launch16<Epi, 1>& l, const Operand16& a, const Operand16& b) {
  if (kind == kPair256) return launch16<psb::Cfg16<2, 256, kPlanes, 2, kLong>, Epi, 1>(chain, l, &a, &b);
  if constexpr (kPlanes == 1 && kLong == 0) {
    if (kind == kPair256Wide) return launch16<psb::Cfg16<2, 256, 1, 4>, Epi, 1>(chain, l, &a, &b);
  }
  if (kind == kPair128) return launch16<psb::Cfg16<2, 128, kPlanes, 2, kLong>, Epi, 1>(chain, l, &a, &b);
  if (kind == kOne128) return launch16<psb::Cfg16<1, 128, kPlanes, 2, kLong>, Epi, 1>(chain, l, &a, &b);
  return launch16<psb::Cfg16<1, 64, kPlanes, 2, kLong>, Epi, 1>(chain, l, &a, &b);
}
template <int kPlanes, class Epi>
int launch_tiled(Chain& chain, int kind, psb::Launch16<Epi, 1>& l, const Operand16& a, const Operand16& b) {
  constexpr int kLong = Epi::kLongK / psb::kG16K;
  if constexpr (kPlanes == 1) {
    if (l.g[0].kb_split > kLong) return launch_kind<1, kLong, Epi>(chain, kind, l, a, b);
  }
  return launch_kind<kPlanes, 0, Epi>(chain, kind, l, a, b);
}
template <class Epi>
int product16(Chain& chain, int planes, int kind, const psb::Gemm16Args& g, const Operand16& a, const Operand16& b, const typename Epi::Params& ep) {
  psb::Launch16<Epi, 1> l = {{g}, {ep}};
  return planes == 2 ? launch_tiled<2, Epi>(chain, kind, l, a, b) : launch_tiled<1, Epi>(chain, kind, l, a, b);
}
// two at once, in tiles of 128x128 or 128x64; sums of up to kLongK
template <class Epi>
int products16(Chain& chain, int planes, int kind, psb::Launch16<Epi, 2>& l, const Operand16* a, const Operand16* b) {
  if (planes == 2)
    return kind == kOne128 ? launch16<psb::Cfg16<1, 128, 2>, Epi, 2>(chain, l, a, b) : launch16<psb::Cfg16<1, 64, 2>, Epi, 2>(chain, l, a, b);
  return kind == kOne128 ? launch16<psb::Cfg16<1, 128, 1>, Epi, 2>(chain, l, a, b) : launch16<psb::Cfg16<1, 64, 1>, Epi, 2>(chain, l, a, b);
}

}  // namespace
