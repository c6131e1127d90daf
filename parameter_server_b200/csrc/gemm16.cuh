// Matrix products of 16-bit operands on the tensor cores with an epilogue of the caller's: D[M,N] = A[M,K] · B[N,K]ᵀ,
// fp32 accumulation in TMEM, one launch for a batch of them.
//
// Operands.  An operand is one 16-bit matrix or, where fp32 accuracy is wanted, two planes of fp16: x·2^s = hi + lo with
// hi = fp16(x·2^s) and lo = fp16(x·2^s − hi), which together carry 22 bits.  The product is then the sum of hi·hi, hi·lo
// and lo·hi in one accumulator; what is left out, lo·lo, is below 2^-22 of the terms.  That costs three 16-bit products
// where three tf32 products (11 bits as well) would cost six.  The tensor cores cut a sum to fp32 at every step of 16
// elements instead of rounding it, an error that grows with the number of steps (K = 60,000: 6e-5 of a gradient); products
// of planes are therefore summed in TMEM for 256 elements of K at a time (48 steps) and added up in the epilogue's
// registers.  An operand may lie either way round in memory: K-major
// ([rows][k], k contiguous) or MN-major ([k][rows], rows contiguous); nothing is transposed in memory.
//
// Shape.  Persistent CTAs, or CTA pairs (cta_group::2) where the problem has enough tiles:
//   warp 0, one lane    TMA producer, a ring of stages of 64 elements of K (128-byte swizzle rows)
//   warp 1, one lane    tcgen05.mma; in a pair the leader issues for both CTAs
//   warps 2-9           epilogue: warp w reads TMEM lanes 32(w % 4)..+31, half of the tile's columns; the accumulator is
//                       double-buffered, so a tile's epilogue runs under the next tile's products
// No load is a multicast.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "psb_tcgen05.cuh"

namespace psb {

constexpr int kG16Threads = 320, kG16K = 64;
constexpr int kG16Smem = 192 * 1024;              // of the stages

template <int kCtas_, int kN_, int kPlanes_, bool kAMN_, bool kBMN_>
struct Cfg16 {
  static constexpr int kCtas = kCtas_, kN = kN_, kPlanes = kPlanes_;
  static constexpr bool kAMN = kAMN_, kBMN = kBMN_;
  static constexpr int kM = 128 * kCtas, kBRows = kN / kCtas;
  static constexpr int kABytes = 128 * 128, kBBytes = kBRows * 128;
  static constexpr int kStageBytes = kPlanes * (kABytes + kBBytes);
  static constexpr int kStages = kG16Smem / kStageBytes > 8 ? 8 : kG16Smem / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 512;
  static constexpr bool kPromote = kPlanes == 2;   // sums of kChunk blocks of K are added up in registers
  static constexpr int kChunk = kPromote ? 4 : 1 << 30;
  static constexpr uint32_t kTmem = 2 * kN < 32 ? 32 : 2 * kN;
  static_assert(kStages >= 3 && kBRows % 64 == 0 && kTmem <= 512, "shape of a tile");
};

struct Gemm16Args {
  CUtensorMap a, b;
  int M, N, K, batch;
  int a_z, b_z;                // matrices of a map per batch entry (planes that lie there, whether read or not); 0: one for all
  int a_m0, a_k0, b_n0, b_k0;  // where the problem starts in the maps
  int splits, kb_split;        // K blocks are dealt to `splits` pieces of kb_split; a piece is a tile of its own
  int sym;                     // square result that is symmetric: only tiles on and above the diagonal
  int bf16;                    // operands are bf16, else fp16
  uint32_t* status;
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

// The dimension with fewer tiles runs fastest: its operand stays in L2 while the other one is read once.
template <class C>
__device__ __forceinline__ Tile16 tile16(const Gemm16Args& g, int t) {
  const int tm = (g.M + C::kM - 1) / C::kM, tn = (g.N + C::kN - 1) / C::kN;
  const int per = g.sym ? tm * (tm + 1) / 2 : tm * tn;
  Tile16 w;
  const int zs = t / per;
  int u = t - zs * per, i, j;
  w.z = zs / g.splits;
  w.split = zs - w.z * g.splits;
  if (g.sym) {
    j = (int)((sqrtf(8.f * (float)u + 1.f) - 1.f) * 0.5f);
    while ((j + 1) * (j + 2) / 2 <= u) ++j;
    while (j * (j + 1) / 2 > u) --j;
    i = u - j * (j + 1) / 2;
  } else if (tm <= tn) {
    i = u % tm; j = u / tm;
  } else {
    j = u % tn; i = u / tn;
  }
  w.mirror = g.sym && i != j;
  w.m0 = i * C::kM; w.n0 = j * C::kN; w.tn = j;
  const int nkb = (g.K + kG16K - 1) / kG16K;
  w.kb0 = w.split * g.kb_split;
  w.kb1 = w.kb0 + g.kb_split < nkb ? w.kb0 + g.kb_split : nkb;
  return w;
}

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
template <int kCtas, bool kMN, int kRows>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, uint32_t bar, int k0, int r0, int z) {
  if constexpr (kMN) {
#pragma unroll
    for (int c = 0; c < kRows / 64; ++c) tma_load_3d<kCtas>(dst + c * 8192, map, bar, r0 + c * 64, k0, z);
  } else {
    tma_load_3d<kCtas>(dst, map, bar, k0, r0, z);
  }
}
// MN-major, 128-byte swizzle: a chunk of 64 rows is 64 k-lines of 128 bytes, 8 lines are a swizzle atom.  Leading
// byte offset (bits 16-29): from a chunk to the next, 8192; stride byte offset: from 8 k-lines to the next, 1024.
template <bool kMN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  uint64_t d = make_smem_desc(addr);
  if (kMN) d |= (uint64_t)(8192 >> 4) << 16;
  return d;
}
// kind::f16: D fp32, A and B fp16 (0) or bf16 (1) at bits 7-9 and 10-12, bits 15 / 16: A / B is MN-major
template <class C>
__device__ __forceinline__ uint32_t idesc16(int bf16) {
  return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | (C::kAMN ? 1u << 15 : 0u) | (C::kBMN ? 1u << 16 : 0u)
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

// An epilogue is a struct with Params, a constructor (params, args, tile, row, half) and
//   chunk(v, col)   32 sums of the row, from column col of the result on (row and col may lie outside)
//   end()           after the last chunk of the row's half tile
template <class C, class Epi>
__global__ void __launch_bounds__(kG16Threads, 1)
gemm16_kernel(const __grid_constant__ Gemm16Args g, const __grid_constant__ typename Epi::Params ep) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + C::kStages * C::kStageBytes);
  uint64_t *empty = full + C::kStages, *tfull = empty + C::kStages, *tempty = tfull + 2;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile uint32_t* abort_flag = tmem_base + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = C::kCtas == 2 ? (int)cluster_rank() : 0;
  const int ntiles = tiles16<C>(g), first = blockIdx.x / C::kCtas, step = gridDim.x / C::kCtas;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], 8 * C::kCtas); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    if constexpr (C::kCtas == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)), "r"(C::kTmem) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)), "r"(C::kTmem) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (C::kCtas == 2) cluster_sync_all();       // the peer's barriers are ready before anything is signalled there
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_base;

  if (warp == 0 && lane == 0) {
    uint32_t it = 0;
    for (int t = first; t < ntiles && !*abort_flag; t += step) {
      const Tile16 w = tile16<C>(g, t);
      const int am = g.a_m0 + w.m0 + rank * 128, bn = g.b_n0 + w.n0 + rank * C::kBRows;
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
        const int st = it % C::kStages;
        if (it >= (uint32_t)C::kStages && !mbar_wait(&empty[st], ((it / C::kStages) - 1) & 1)) { *abort_flag = 1; break; }
        if (rank == 0) mbar_expect_tx(&full[st], C::kCtas * C::kStageBytes);
        const uint32_t bar = C::kCtas == 2 ? mapa_u32(smem_u32(&full[st]), 0) : smem_u32(&full[st]);
        const uint32_t sa = smem_u32(stages + st * C::kStageBytes), sb = sa + C::kPlanes * C::kABytes;
#pragma unroll
        for (int p = 0; p < C::kPlanes; ++p) {
          load_operand<C::kCtas, C::kAMN, 128>(sa + p * C::kABytes, &g.a, bar, g.a_k0 + kb * kG16K, am, w.z * g.a_z + p);
          load_operand<C::kCtas, C::kBMN, C::kBRows>(sb + p * C::kBBytes, &g.b, bar, g.b_k0 + kb * kG16K, bn, w.z * g.b_z + p);
        }
      }
    }
    // the last releases must have landed here before this CTA's shared memory may go away
    for (uint32_t u = it > (uint32_t)C::kStages ? it - C::kStages : 0; u < it && !*abort_flag; ++u)
      if (!mbar_wait(&empty[u % C::kStages], (u / C::kStages) & 1)) *abort_flag = 1;
  } else if (warp == 1 && lane == 0 && rank == 0) {
    const uint32_t idesc = idesc16<C>(g.bf16);
    uint32_t it = 0, n = 0;
    for (int t = first; t < ntiles && !*abort_flag; t += step) {
      const Tile16 w = tile16<C>(g, t);
      for (int kc = w.kb0; kc < w.kb1 && !*abort_flag; kc += C::kChunk, ++n) {
        const uint32_t acc = n & 1u;
        if (n >= 2 && !mbar_wait(&tempty[acc], ((n >> 1) - 1) & 1)) { *abort_flag = 1; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + acc * (uint32_t)C::kN;
        const int ke = w.kb1 - kc < C::kChunk ? w.kb1 : kc + C::kChunk;
        uint32_t accumulate = 0;
        for (int kb = kc; kb < ke; ++kb, ++it) {
          const int st = it % C::kStages;
          if (!mbar_wait(&full[st], (it / C::kStages) & 1)) { *abort_flag = 1; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sa = smem_u32(stages + st * C::kStageBytes), sb = sa + C::kPlanes * C::kABytes;
#pragma unroll
          for (int q = 0; q < (C::kPlanes == 2 ? 3 : 1); ++q) {      // hi·lo, lo·hi, hi·hi
            const uint64_t da = operand_desc<C::kAMN>(sa + (q == 1 ? C::kABytes : 0));
            const uint64_t db = operand_desc<C::kBMN>(sb + (C::kPlanes == 2 && q == 0 ? C::kBBytes : 0));
#pragma unroll
            for (int k = 0; k < kG16K / 16; ++k) {     // 16 elements of K: 32 bytes of a K-major row, 16 MN-major lines
              mma16<C::kCtas>(d, da + (uint64_t)(k * (C::kAMN ? 2048 : 32) >> 4), db + (uint64_t)(k * (C::kBMN ? 2048 : 32) >> 4), idesc, accumulate);
              accumulate = 1;
            }
          }
          commit16<C::kCtas>(&empty[st]);
        }
        commit16<C::kCtas>(&tfull[acc]);
      }
    }
  } else if (warp >= 2) {
    constexpr int kHalf = C::kN / 2;
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * kHalf);
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
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapa_u32(smem_u32(&tempty[acc]), 0)) : "memory");
        else
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&tempty[acc])) : "memory");
      }
    };
    bool ok = true;
    for (int t = first; t < ntiles && ok; t += step) {
      const Tile16 w = tile16<C>(g, t);
      const int row = w.m0 + rank * 128 + q * 32 + lane, col = w.n0 + half * kHalf;
      if constexpr (C::kPromote) {
        float sum[kHalf];
        for (int kc = w.kb0; kc < w.kb1; kc += C::kChunk, ++n) {
          const uint32_t acc = n & 1u;
          if (!(ok = sums_ready(acc, (n >> 1) & 1))) break;
#pragma unroll
          for (int c = 0; c < kHalf; c += 32) {
            uint32_t r[32];
            tmem_load_32x32(lanes + acc * (uint32_t)C::kN + (uint32_t)c, r);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[c + j] = kc == w.kb0 ? __uint_as_float(r[j]) : sum[c + j] + __uint_as_float(r[j]);
          }
          release(acc);
        }
        if (!ok) break;
        Epi epi(ep, g, w, row, half);
#pragma unroll
        for (int c = 0; c < kHalf; c += 32) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = sum[c + j];
          epi.chunk(v, col + c);
        }
        epi.end();
      } else {
        const uint32_t acc = n & 1u;
        if (!(ok = sums_ready(acc, (n >> 1) & 1))) break;
        ++n;
        Epi epi(ep, g, w, row, half);
#pragma unroll 1
        for (int c = 0; c < kHalf; c += 32) {
          uint32_t r[32];
          tmem_load_32x32(lanes + acc * (uint32_t)C::kN + (uint32_t)c, r);
          tmem_load_wait();
          if (c + 32 >= kHalf) release(acc);
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          epi.chunk(v, col + c);
        }
        epi.end();
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) set_status(g.status, kWaitTimeout, blockIdx.x, 400);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (C::kCtas == 2) cluster_sync_all();       // neither CTA frees its accumulators or leaves while the other still works
  if (warp == 0) {
    if constexpr (C::kCtas == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
  }
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
// the box is 64 columns of box_rows rows.  0, a driver error, or -1 without the driver's entry point.
int make_map16(CUtensorMap* map, const void* base, int bf16, int64_t rows, int64_t cols, int64_t ld, int64_t stride, int count, int box_rows) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return -1;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(count > 1 ? stride : ld * rows) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
  return (int)enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box,
                  estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// One 16-bit matrix, or `planes` of them `plane_stride` elements apart per batch entry, as a caller describes it
struct Operand16 {
  const void* base;
  int64_t rows, cols, ld, stride;     // of the memory: rows of `cols` contiguous elements
  int count;                          // matrices in the map
};

template <class C, class Epi>
int launch16(psb::Gemm16Args g, const Operand16& a, const Operand16& b, const typename Epi::Params& ep, cudaStream_t stream) {
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms <= 0) return (int)cudaErrorInvalidDevice;
  int r = make_map16(&g.a, a.base, g.bf16, a.rows, a.cols, a.ld, a.stride, a.count, C::kAMN ? 64 : 128);
  if (r == 0) r = make_map16(&g.b, b.base, g.bf16, b.rows, b.cols, b.ld, b.stride, b.count, C::kBMN ? 64 : C::kBRows);
  if (r) return r;
  static bool attr[kMaxDevices] = {};
  if (!attr[dev]) {
    cudaError_t e = cudaFuncSetAttribute(psb::gemm16_kernel<C, Epi>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return (int)e;
    attr[dev] = true;
  }
  const int tiles = psb::tiles16<C>(g), most = sms / C::kCtas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((tiles < most ? tiles : most) * C::kCtas));
  cfg.blockDim = dim3(psb::kG16Threads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C::kCtas; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C::kCtas == 2 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, psb::gemm16_kernel<C, Epi>, g, ep);
}

}  // namespace
