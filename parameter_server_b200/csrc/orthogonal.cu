// Orthogonalised weight updates: Newton-Schulz steps on the tensor cores (gemm16.cuh).
//
//   X = U / (|U|_F + eps);   `steps` times:  A = X Xᵀ,  X ← a X + (b A + c A²) X        on the shorter side of X
//
// with the odd polynomial of the Muon optimiser, (a, b, c) = (3.4445, −4.7750, 2.0315), which brings every singular value
// of X into about [0.7, 1.2].  For the update U = g + μ m (Nesterov) or m after m ← μ m + g, and w ← w − lr X at the end.
//
// A step is three products.  A and b A + c A² are symmetric: only the tiles on and above the diagonal are made, a tile
// above it is stored a second time, transposed.  The linear terms are on the diagonals of the factors (EpiNs), so that no
// product reads a third matrix.  A matrix that is taller than wide is not transposed: A = Xᵀ X reads X
// MN-major, and X (a I + b A + c A²) reads the symmetric factor either way.  Scale and step of the weights are in the last
// product's epilogue.
//
// Precision.  No entry of X, A or b A + c A² exceeds 12 in magnitude (singular values of X stay below 1.3), so all are
// kept times 2^10 in fp16, as two planes (22 bits) or one (11).  A rounding made in step k is multiplied by up to a = 3.44
// in every later step where it falls on small singular values: with one plane throughout, a matrix of a few strong
// directions over weak noise (ratio 10^2 and more) comes out 4 % off, which 16-bit results show.  bf16 results take one plane
// in the last step only, which leaves 0.05 to 0.12 % (they are rounded to 0.17 % on average); fp32 and fp16 results take
// two throughout (8e-6 for the same matrix, 3e-7 for a random one).
//
// 4096 x 4096, bf16: 3.2 ms for 1.37 TFLOP (symmetric products in halves), 3.57 with the products of planes, which take 2.1 ms
// at the rate of a plain cuBLAS product.  Tiles come in whole rounds of 74 pairs, and a round ends with an epilogue of two planes.
#include "gemm16.cuh"

namespace psb {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kNsScale = 1024.f, kNsInv = 1.f / 1024.f;
constexpr int kNormBlocks = 592;

enum : int { kOrthF32 = 0, kOrthBF16 = 1, kOrthF16 = 2 };

struct OrthArgs {
  const void* x;               // the matrix, or the gradient of an update; [batch][rows][cols]
  float* m;                    // momentum of an update (updated), else null
  void* out;                   // the result, or the fp32 weights of an update (updated)
  int batch, rows, cols, dtype, steps, nesterov;
  float lr, momentum, eps, pad;
  void* ws;
  int64_t ws_bytes;
  uint32_t* status;
};

__device__ __forceinline__ float load_as(const void* p, int64_t at, int dtype) {
  if (dtype == kOrthF32) return reinterpret_cast<const float*>(p)[at];
  if (dtype == kOrthBF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[at]);
  return __half2float(reinterpret_cast<const __half*>(p)[at]);
}
__device__ __forceinline__ float update_direction(float g, float m, float mu, int nesterov) { return nesterov ? g + mu * m : m; }

// Four neighbours from an address that is aligned to them
__device__ __forceinline__ float4 load4_as(const void* p, int64_t at, int dtype) {
  if (dtype == kOrthF32) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
  const uint2 t = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + at);
  if (dtype == kOrthBF16) {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&t.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&t.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// Momentum, and the squares of U summed in fp64 (a gradient's entries may be anywhere in fp32's range), a block's sum each.
// Bound by HBM; with four times four elements of a thread on their way (one at a time: 1024 x 4096 with momentum, 50 MB,
// 33 us; so 11.6).
__global__ void __launch_bounds__(256)
k_orth_norm(const void* __restrict__ x, float* __restrict__ m, int64_t numel, int dtype, float mu, int nesterov, double* __restrict__ part) {
  pdl_wait();
  const int64_t base = (int64_t)blockIdx.y * numel, step = (int64_t)gridDim.x * 256;
  const bool fours = ((numel & 3) | (reinterpret_cast<uintptr_t>(m) & 15) | (reinterpret_cast<uintptr_t>(x) & (dtype == kOrthF32 ? 15 : 7))) == 0;
  double acc = 0.0;
  if (fours) {
    const int64_t n4 = numel / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += 4 * step) {
      float4 u[4], v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (i + k * step >= n4) break;
        const int64_t at = base + (i + k * step) * 4;
        u[k] = load4_as(x, at, dtype);
        if (m != nullptr) v[k] = *reinterpret_cast<const float4*>(m + at);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (i + k * step >= n4) break;
        float e[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
        if (m != nullptr) {
          float t[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            t[j] = mu * t[j] + e[j];
            e[j] = update_direction(e[j], t[j], mu, nesterov);
          }
          *reinterpret_cast<float4*>(m + base + (i + k * step) * 4) = make_float4(t[0], t[1], t[2], t[3]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc += (double)e[j] * e[j];
      }
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += step) {
      float u = load_as(x, base + i, dtype);
      if (m != nullptr) {
        const float mv = mu * m[base + i] + u;
        m[base + i] = mv;
        u = update_direction(u, mv, mu, nesterov);
      }
      acc += (double)u * u;
    }
  }
  __shared__ double sh[8];
  acc = warp_sum_d(acc);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < 8; ++i) t += sh[i];
    part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = t;
  }
}

__device__ __forceinline__ void planes8(const float* v, uint4& h, uint4& l) {
  uint32_t hs[4], ls[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hs[i] = pair16<kFmtPlanes>(v[2 * i], v[2 * i + 1], false);
    ls[i] = pair16<kFmtPlanes>(v[2 * i], v[2 * i + 1], true);
  }
  h = make_uint4(hs[0], hs[1], hs[2], hs[3]);
  l = make_uint4(ls[0], ls[1], ls[2], ls[3]);
}

// U / (|U| + eps) into the planes
__global__ void __launch_bounds__(256)
k_orth_pack(const void* __restrict__ x, const float* m, int rows, int cols, int dtype, float mu, int nesterov, const double* part,
            int nparts, float eps, uint16_t* __restrict__ out, int64_t ld, int64_t plane) {
  __shared__ double sh[8];
  pdl_wait();
  const int64_t base = (int64_t)blockIdx.y * rows * cols;
  double t = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) t += part[(int64_t)blockIdx.y * nparts + i];
  t = warp_sum_d(t);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = t;
  __syncthreads();
  t = 0.0;
  for (int i = 0; i < 8; ++i) t += sh[i];
  const double f = (double)kNsScale / (sqrt(t) + (double)eps);
  uint16_t* dst = out + (int64_t)blockIdx.y * 2 * plane;
  // rows without padding are one long row: eights of it, two at a time
  if (ld == cols && ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(x)) & 15) == 0) {
    const int64_t eights = (int64_t)rows * cols / 8, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < eights; i += 2 * step) {
      float4 u[2][2], v[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (i + k * step >= eights) break;
        const int64_t at = base + (i + k * step) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u[k][h] = load4_as(x, at + 4 * h, dtype);
          if (m != nullptr) v[k][h] = *reinterpret_cast<const float4*>(m + at + 4 * h);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (i + k * step >= eights) break;
        float e[8] = {u[k][0].x, u[k][0].y, u[k][0].z, u[k][0].w, u[k][1].x, u[k][1].y, u[k][1].z, u[k][1].w};
        const float t[8] = {v[k][0].x, v[k][0].y, v[k][0].z, v[k][0].w, v[k][1].x, v[k][1].y, v[k][1].z, v[k][1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = (float)((double)(m != nullptr ? update_direction(e[j], t[j], mu, nesterov) : e[j]) * f);
        uint4 h, l;
        planes8(e, h, l);
        *reinterpret_cast<uint4*>(dst + (i + k * step) * 8) = h;
        *reinterpret_cast<uint4*>(dst + plane + (i + k * step) * 8) = l;
      }
    }
    return;
  }
  const int per = (int)(ld / 2);
  const int64_t total = (int64_t)rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 2;
    __half h[2], l[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float u = 0.f;
      if (c + j < cols) {
        const int64_t at = base + r * cols + c + j;
        u = load_as(x, at, dtype);
        if (m != nullptr) u = update_direction(u, m[at], mu, nesterov);
      }
      // f may lie outside fp32 where U is tiny or huge; the quotient does not
      split16((float)((double)u * f), h[j], l[j]);
    }
    *reinterpret_cast<uint32_t*>(dst + r * ld + c) = pack_half2(h[0], h[1]);
    *reinterpret_cast<uint32_t*>(dst + plane + r * ld + c) = pack_half2(l[0], l[1]);
  }
}

// alpha · product + beta · I, to planes (and transposed where the tile has a mirror image), to fp32 slots of a split K, to the
// result, or as a step of the weights.  For A, a second matrix alpha2 · product + beta2 · I: b I + c A, so that
// b A + c A² + a I = A (b I + c A) + a I and the new X = (a I + b A + c A²) X are plain products.
__host__ __device__ __forceinline__ int up4(int n) { return (n + 3) & ~3; }
struct EpiNs {
  static constexpr int kLongK = 32768;
  struct Params {
    CUtensorMap out[2];
    float* slots;              // not null: raw sums, [split][batch][M][N rounded up to fours]
    void* result;              // not null: the last product
    int M, N, batch, second, dtype, update;
    float alpha, beta, alpha2, beta2, lr;
  };
  template <int kPart>
  static __device__ __forceinline__ void ahead(const Params& p, const Tile16& w, int row, int col, int lane) {
    if (p.update && row + lane < p.M) prefetch_l2<kPart>(reinterpret_cast<const float*>(p.result) + ((int64_t)w.z * p.M + row + lane) * p.N, col, p.N);
  }
  template <int kPlanes, int kPart, class Stage, class Sums, class Done>
  static __device__ __forceinline__ void run(const Params& p, const Gemm16Args&, const Tile16& w, int row0, int col0, int, Stage& st,
                                             const Sums& sums, Done done) {
    constexpr int kFmt = kPlanes == 2 ? kFmtPlanes : kFmtF16;
#pragma unroll 1
    for (int k = 0; k < kPart; k += 32) {
      float v[32];
      sums.load(k, v);
      if (k + 32 >= kPart) done();
      const int col = col0 + k;
      if (row0 >= p.M || col >= p.N) continue;
      if (p.slots == nullptr && p.result == nullptr) {
        const bool diagonal = row0 == col;                 // both are multiples of 32
#pragma unroll 1
        for (int m = 0; m < (p.second ? 2 : 1); ++m) {
          const float alpha = m ? p.alpha2 : p.alpha, beta = m ? p.beta2 : p.beta;
          float u[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) u[j] = alpha * v[j] + (diagonal && j == st.lane ? beta : 0.f);
          st.template store<kFmt>(&p.out[m], u, row0, col, w.z * 2, w.mirror);
        }
        continue;
      }
      const int rows = p.M - row0 < 32 ? p.M - row0 : 32, mine = col + st.lane;
      const bool in = mine < p.N;
      st.by_rows(v, [&](auto value) {
        if (!in) return;
        if (p.slots != nullptr) {
          const int ld = up4(p.N);
          float* dst = p.slots + (((int64_t)w.split * p.batch + w.z) * p.M + row0) * ld + mine;
#pragma unroll 8
          for (int r = 0; r < rows; ++r, dst += ld) *dst = value(r);
          return;
        }
        const int64_t at = ((int64_t)w.z * p.M + row0) * p.N + mine;
        const float f = p.alpha * kNsInv;
        if (!p.update) {
          if (p.dtype == kOrthF32) {
            float* dst = reinterpret_cast<float*>(p.result) + at;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, dst += p.N) *dst = f * value(r);
          } else if (p.dtype == kOrthBF16) {
            __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.result) + at;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, dst += p.N) *dst = __float2bfloat16_rn(f * value(r));
          } else {
            __half* dst = reinterpret_cast<__half*>(p.result) + at;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, dst += p.N) *dst = __float2half_rn(f * value(r));
          }
          return;
        }
        float* wt = reinterpret_cast<float*>(p.result) + at;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 16) {
          float t[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) t[i] = r0 + i < rows ? wt[(int64_t)(r0 + i) * p.N] : 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (r0 + i < rows) wt[(int64_t)(r0 + i) * p.N] = t[i] - p.lr * (f * value(r0 + i));
        }
      });
    }
  }
};

// The splits of a product's K to planes: alpha · sum + beta · I, and the second matrix.  Of a symmetric product only the
// tiles (tile x tile) on and above the diagonal exist (tile 0: all do).  A block takes 32 x 32, a thread four neighbours, and stores them
// and, through shared memory, their transpose.  Rows of the sums start at 16 bytes whatever n is (9 pieces of 461 x 461: 8.3 us with
// loads of single floats, 6.9 so).
__global__ void __launch_bounds__(256)
k_orth_sum(const float* slots, int splits, int batch, int n, int tile, uint16_t* __restrict__ out, uint16_t* __restrict__ out2,
           int64_t ld, int64_t plane, float alpha, float beta, float alpha2, float beta2) {
  __shared__ float sum[32][33];
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32, z = blockIdx.z;
  if (tile > 0 && r0 / tile > c0 / tile) return;
  const bool twice = tile > 0 && r0 / tile < c0 / tile;
  pdl_wait();
  const int ty = threadIdx.x >> 3, tx = (threadIdx.x & 7) * 4;
  const int64_t per = (int64_t)n * up4(n), total = per * batch, base = (int64_t)z * 2 * plane;
  const float* src = slots + z * per + (int64_t)(r0 + ty) * up4(n) + c0 + tx;
  float v[4] = {};
  if (r0 + ty < n && c0 + tx < n) {
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      const float4 t = *reinterpret_cast<const float4*>(src + s * total);
      v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
    }
  }
  // four elements of row r from column c on; rows are padded to 8 elements and what lies behind their end is not read
  auto put = [&](int r, int c, const float (&x)[4]) {
    const int64_t at = base + (int64_t)r * ld + c;
    uint2 h, l;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (m == 1 && out2 == nullptr) break;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = (m ? alpha2 : alpha) * x[j] + (r == c + j ? (m ? beta2 : beta) : 0.f);
      h = make_uint2(pair16<kFmtPlanes>(y[0], y[1], false), pair16<kFmtPlanes>(y[2], y[3], false));
      l = make_uint2(pair16<kFmtPlanes>(y[0], y[1], true), pair16<kFmtPlanes>(y[2], y[3], true));
      *reinterpret_cast<uint2*>((m ? out2 : out) + at) = h;
      *reinterpret_cast<uint2*>((m ? out2 : out) + at + plane) = l;
    }
  };
  if (r0 + ty < n && c0 + tx < n) put(r0 + ty, c0 + tx, v);
  if (!twice) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[ty][tx + j] = v[j];
  __syncthreads();
  const float t[4] = {sum[tx][ty], sum[tx + 1][ty], sum[tx + 2][ty], sum[tx + 3][ty]};       // column ty, a row of the mirror image
  if (c0 + ty < n && r0 + tx < n) put(c0 + ty, r0 + tx, t);
}

// ------------------------------------------------------------------ matrices that fit into shared memory
// A matrix whose shorter side is at most 128 stays on the SMs for all of its steps: a cluster of CTAs holds it, each a slice
// of the longer side, and each the whole of the small squares.  One launch instead of 17, of which each costs 6 us however
// small it is.  Operands lie in shared memory as the tensor cores read them: X [lo][slice] in swizzled rows of 64 columns,
// which is K-major for X Xᵀ and, the same bytes, MN-major for B X.
//   X Xᵀ of the slice -> fp32 sums; a share of them is added up over the CTAs (in their order) and sent to all, as planes
//   B = A (b I + c A) + a I by every CTA for itself; X = B X of the slice
// Two planes throughout.  A product this small takes the tensor cores some 80 cycles whatever its width, so hi·hi and
// hi·lo are one product: the planes of 64 columns lie behind one another, and rows of both are the N of one instruction.
// Sums over more than 128 columns have an accumulator for each 128.
struct SmallArgs {
  OrthArgs o;
  int lo, hi, tall, lop, hs, cl;               // lop: lo in 16s, hs: width of a slice in 64s, cl: CTAs of a cluster
  int a_off, a2_off, p_off;
};
constexpr int kSmallThreads = 512, kSmallParts = kSmallThreads / 128;

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_own_v4(uint32_t addr, uint4 v) {
  asm volatile("st.shared::cta.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float4 ld_own_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cta.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// Byte offset of eight columns (the c8-th eight) of a row in an operand of `rows` rows: blocks of 64 columns, the hi and then
// the lo plane of each.
__device__ __forceinline__ uint32_t tile_at(int row, int c8, int rows) {
  return (uint32_t)((c8 >> 3) * rows * 256 + row * 128 + (((c8 & 7) ^ (row & 7)) << 4));
}

__global__ void __launch_bounds__(kSmallThreads, 1)
k_orth_small(const __grid_constant__ SmallArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t done;
  __shared__ uint32_t tmem_base, abort_flag;
  __shared__ double sums[16], shared_sum[kSmallThreads / 32];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, q = warp & 3, part = warp >> 2;
  const int rank = p.cl > 1 ? (int)cluster_rank() : 0, z = blockIdx.x / p.cl;
  const int lo = p.lo, lop = p.lop, hs = p.hs, c0 = rank * hs, width = p.hi - c0 < 0 ? 0 : p.hi - c0 < hs ? p.hi - c0 : hs;
  const uint32_t X = smem_u32(base), A = smem_u32(base + p.a_off), A2 = smem_u32(base + p.a2_off), P = smem_u32(base + p.p_off);
  const uint32_t lo_plane = (uint32_t)(lop * 128);          // from a hi to its lo plane

  if (tid == 0) {
    mbar_init(&done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();

  // Momentum, norm, and U in fp32 at X's place: eight columns of a row take the bytes of their two planes.  Consecutive
  // threads go along what is contiguous in memory; the next eight are on their way while these are worked on.
  const int64_t at0 = (int64_t)z * p.o.rows * p.o.cols;
  const int per_row = hs / 8, eights = lop * per_row;
  const bool moving = p.o.m != nullptr;
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.o.x) | reinterpret_cast<uintptr_t>(p.o.m);
  const bool vec = !p.tall && p.o.dtype == kOrthF32 && (p.hi & 3) == 0 && (all & 15) == 0;
  struct Eight { int r, c8, left; int64_t at; float u[8], m[8]; };
  const int64_t by = p.tall ? lo : 1;
  auto fetch = [&](int i, Eight& e) {
    e.r = p.tall ? i % lop : i / per_row;
    e.c8 = p.tall ? i / lop : i % per_row;
    e.left = i < eights && e.r < lo ? width - e.c8 * 8 : 0;
    e.at = at0 + (p.tall ? (int64_t)(c0 + e.c8 * 8) * lo + e.r : (int64_t)e.r * p.hi + c0 + e.c8 * 8);
    if (vec && e.left >= 8) {
      const float4* xs = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.o.x) + e.at);
      *reinterpret_cast<float4*>(e.u) = xs[0];
      *reinterpret_cast<float4*>(e.u + 4) = xs[1];
      if (moving) {
        *reinterpret_cast<float4*>(e.m) = *reinterpret_cast<const float4*>(p.o.m + e.at);
        *reinterpret_cast<float4*>(e.m + 4) = *reinterpret_cast<const float4*>(p.o.m + e.at + 4);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e.u[j] = j < e.left ? load_as(p.o.x, e.at + j * by, p.o.dtype) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) e.m[j] = moving && j < e.left ? p.o.m[e.at + j * by] : 0.f;
    }
  };
  double acc = 0.0;
  Eight next;
  fetch(tid, next);
  for (int i = tid; i < eights; i += kSmallThreads) {
    Eight e = next;
    fetch(i + kSmallThreads, next);
    if (moving) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e.m[j] = p.o.momentum * e.m[j] + e.u[j];
        e.u[j] = update_direction(e.u[j], e.m[j], p.o.momentum, p.o.nesterov);
      }
      if (vec && e.left >= 8) {
        *reinterpret_cast<float4*>(p.o.m + e.at) = *reinterpret_cast<float4*>(e.m);
        *reinterpret_cast<float4*>(p.o.m + e.at + 4) = *reinterpret_cast<float4*>(e.m + 4);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < e.left) p.o.m[e.at + j * by] = e.m[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc += (double)e.u[j] * e.u[j];
    const uint32_t to = X + tile_at(e.r, e.c8, lop);
    st_own_v4(to, *reinterpret_cast<uint4*>(e.u));
    st_own_v4(to + lo_plane, *reinterpret_cast<uint4*>(e.u + 4));
  }
  acc = warp_sum_d(acc);
  if (lane == 0) shared_sum[warp] = acc;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
  double total = 0.0;
  for (int i = 0; i < kSmallThreads / 32; ++i) total += shared_sum[i];
  if (p.cl > 1) {
    cluster_sync_all();                                   // every CTA runs
    if (tid < p.cl)
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_u32(smem_u32(&sums[rank]), (uint32_t)tid)), "d"(total) : "memory");
    cluster_sync_all();
    total = 0.0;
    for (int i = 0; i < p.cl; ++i) total += sums[i];
  }
  const double f = (double)kNsScale / (sqrt(total) + (double)p.o.eps);
  for (int i = tid; i < eights; i += kSmallThreads) {      // this thread's own
    const uint32_t to = X + (p.tall ? tile_at(i % lop, i / lop, lop) : tile_at(i / per_row, i % per_row, lop));
    const float4 a = ld_own_v4(to), b = ld_own_v4(to + lo_plane);
    const float u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)((double)u[j] * f);      // f may lie outside fp32 where U is tiny or huge
    uint4 h, l;
    planes8(v, h, l);
    st_own_v4(to, h);
    st_own_v4(to + lo_plane, l);
  }

  uint32_t phase = 0;
  auto finish_products = [&] {                             // by warp 0, which issues the products
    if (elect_one()) asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&done)) : "memory");
  };
  auto wait_products = [&] {
    if (lane == 0 && abort_flag == 0 && !mbar_wait(&done, phase & 1)) abort_flag = 1;
    ++phase;
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  auto operands_ready = [&] {                              // written by all threads, read by the tensor cores next
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  // 16 sums of this lane's row from a column on, from two accumulators, or more where stride is given
  const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
  auto add16 = [&](float (&v)[16], uint32_t column) {
    uint32_t r[16];
    __syncwarp();                                          // half of the lanes may have left the turn before
    tmem_load_32x16(lanes + column, r);
    tmem_load_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] += __uint_as_float(r[j]);
  };
  // N = rows of both planes, or of one
  const uint32_t idesc_both = (1u << 4) | ((uint32_t)(2 * lop >> 3) << 17) | (8u << 24), idesc_one = (1u << 4) | ((uint32_t)(lop >> 3) << 17) | (8u << 24);
  const uint64_t lo_off = (uint64_t)(lo_plane >> 4), block = (uint64_t)(uint32_t)(lop * 16);      // in units of 16 bytes
  const int row = q * 32 + lane, groups = (hs + 127) / 128;
  const bool busy = q * 32 < lop;                          // this warp's lanes hold rows
  operands_ready();

  for (int step = 0; step < p.o.steps; ++step) {
    // ---- X Xᵀ of the slice, for each 128 columns: hi·hi in lop columns of TMEM, hi·lo + lo·hi in the next lop
    if (warp == 0) {
      const uint64_t x = make_smem_desc(X);
      for (int g = 0; g < groups; ++g) {
        const uint32_t d = tmem + (uint32_t)(g * 2 * lop);
        uint32_t accumulate = 0;
        for (int ch = 2 * g; ch < 2 * g + 2 && ch * 64 < hs; ++ch) {
          const uint64_t at = x + (uint64_t)(uint32_t)ch * block;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16<1>(d, at + 2 * k, at + 2 * k, idesc_both, k == 0 ? accumulate : 1u);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16<1>(d + (uint32_t)lop, at + lo_off + 2 * k, at + 2 * k, idesc_one, 1u);
          }
          accumulate = 1;
        }
      }
      finish_products();
    }
    __syncwarp();
    wait_products();
    if (busy)
      for (int u = part; u < lop / 16; u += kSmallParts) {
        float v[16] = {};
        for (int g = 0; g < 2 * groups; ++g) add16(v, (uint32_t)(g * lop + u * 16));
        if (row >= lop) continue;
        if (p.cl > 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) st_own_v4(P + (uint32_t)(row * lop * 4 + (((u * 4 + j) ^ (row & 3)) << 4)), *reinterpret_cast<uint4*>(v + 4 * j));
          continue;
        }
        float b[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] *= kNsInv;
          b[j] = kNsC * v[j] + (row == u * 16 + j ? kNsB * kNsScale : 0.f);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4 h, l;
          const uint32_t at = tile_at(row, u * 2 + e, lop);
          planes8(v + 8 * e, h, l);
          st_own_v4(A + at, h);
          st_own_v4(A + at + lo_plane, l);
          planes8(b + 8 * e, h, l);
          st_own_v4(A2 + at, h);
          st_own_v4(A2 + at + lo_plane, l);
        }
      }
    if (p.cl > 1) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      cluster_sync_all();
      const int units = lop * lop / 8, per = (units + p.cl - 1) / p.cl;
      for (int i = rank * per + tid; i < (rank + 1) * per && i < units; i += kSmallThreads) {
        const int r = i / (lop / 8), c8 = i % (lop / 8);
        float v[8] = {}, b[8];
        for (int s = 0; s < p.cl; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 t = ld_cluster_v4(mapa_u32(P + (uint32_t)(r * lop * 4 + (((c8 * 2 + e) ^ (r & 3)) << 4)), (uint32_t)s));
            v[4 * e] += t.x; v[4 * e + 1] += t.y; v[4 * e + 2] += t.z; v[4 * e + 3] += t.w;
          }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] *= kNsInv;
          b[j] = kNsC * v[j] + (r == c8 * 8 + j ? kNsB * kNsScale : 0.f);
        }
        uint4 ah, al, bh, bl;
        planes8(v, ah, al);
        planes8(b, bh, bl);
        const uint32_t at = tile_at(r, c8, lop);
        for (int s = 0; s < p.cl; ++s) {
          const uint32_t to = mapa_u32(A + at, (uint32_t)s), to2 = mapa_u32(A2 + at, (uint32_t)s);
          st_cluster_v4(to, ah);
          st_cluster_v4(to + lo_plane, al);
          st_cluster_v4(to2, bh);
          st_cluster_v4(to2 + lo_plane, bl);
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");
      cluster_sync_all();
    }
    operands_ready();

    // ---- B = A (b I + c A) + a I, into A's place
    if (warp == 0) {
      const uint64_t a = make_smem_desc(A), a2 = make_smem_desc(A2);
      for (int ch = 0; ch * 64 < lop; ++ch) {
        const uint64_t off = (uint64_t)(uint32_t)ch * block;
        const int ks = lop - ch * 64 < 64 ? (lop - ch * 64) / 16 : 4;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < ks) mma16<1>(tmem, a + off + 2 * k, a2 + off + 2 * k, idesc_both, ch > 0 || k > 0 ? 1u : 0u);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < ks) mma16<1>(tmem + (uint32_t)lop, a + off + lo_off + 2 * k, a2 + off + 2 * k, idesc_one, 1u);
        }
      }
      finish_products();
    }
    __syncwarp();
    wait_products();
    if (busy)
      for (int u = part; u < lop / 16; u += kSmallParts) {
        float v[16] = {};
        add16(v, (uint32_t)(u * 16));
        add16(v, (uint32_t)(lop + u * 16));
        if (row >= lop) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = kNsInv * v[j] + (row == u * 16 + j ? kNsA * kNsScale : 0.f);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4 h, l;
          const uint32_t at = tile_at(row, u * 2 + e, lop);
          planes8(v + 8 * e, h, l);
          st_own_v4(A + at, h);
          st_own_v4(A + at + lo_plane, l);
        }
      }
    operands_ready();

    // ---- X = B X of the slice; X is MN-major here: blocks of 64 columns, lop lines of the hi plane and as many of the lo.
    // Up to 128 columns both planes are one N (their blocks take turns in TMEM), beyond that N is wide enough.
    const bool both = hs <= 128;
    if (warp == 0) {
      const uint64_t b = make_smem_desc(A), x = make_smem_desc(X), plane_lead = (uint64_t)((lop * 128) >> 4) << 16, block_lead = plane_lead << 1;
      for (int n0 = 0; n0 < hs; n0 += 256) {
        const int n = hs - n0 < 256 ? hs - n0 : 256;
        const uint32_t mn = (1u << 4) | (1u << 16) | (8u << 24), one = mn | ((uint32_t)(n >> 3) << 17), two = mn | ((uint32_t)(2 * n >> 3) << 17);
        const uint64_t at = x + (uint64_t)(uint32_t)(n0 / 64) * block;
        for (int ch = 0; ch * 64 < lop; ++ch) {
          const uint64_t off = b + (uint64_t)(uint32_t)ch * block, lines = (uint64_t)(uint32_t)(ch * 512);       // 64 lines
          const int ks = lop - ch * 64 < 64 ? (lop - ch * 64) / 16 : 4;
          if (elect_one()) {
            if (both) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < ks) mma16<1>(tmem, off + 2 * k, (at + lines + 128 * k) | plane_lead, two, ch > 0 || k > 0 ? 1u : 0u);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < ks) mma16<1>(tmem + (uint32_t)(2 * hs), off + lo_off + 2 * k, (at + lines + 128 * k) | block_lead, one, ch > 0 || k > 0 ? 1u : 0u);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < ks) mma16<1>(tmem + (uint32_t)n0, off + 2 * k, (at + lo_off + lines + 128 * k) | block_lead, one, ch > 0 || k > 0 ? 1u : 0u);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < ks) mma16<1>(tmem + (uint32_t)n0, off + lo_off + 2 * k, (at + lines + 128 * k) | block_lead, one, 1u);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < ks) mma16<1>(tmem + (uint32_t)n0, off + 2 * k, (at + lines + 128 * k) | block_lead, one, 1u);
            }
          }
        }
      }
      finish_products();
    }
    __syncwarp();
    wait_products();
    const bool last = step + 1 == p.o.steps;
    if (busy)
      for (int u = part; u < hs / 16; u += kSmallParts) {
        float v[16] = {};
        if (both) {
          const uint32_t at = (uint32_t)((u >> 2) * 128 + (u & 3) * 16);
          add16(v, at);
          add16(v, at + 64);
          add16(v, (uint32_t)(2 * hs + u * 16));
        } else {
          add16(v, (uint32_t)(u * 16));
        }
        if (row >= lop) continue;
        if (!last) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] *= kNsInv;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint4 h, l;
            const uint32_t at = tile_at(row, u * 2 + e, lop);
            planes8(v + 8 * e, h, l);
            st_own_v4(X + at, h);
            st_own_v4(X + at + lo_plane, l);
          }
          continue;
        }
        // the result in fp32 over X (and, by a column of each row, A): as it lies in memory, for all threads to store
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] *= kNsInv * kNsInv;
        if (p.tall) {
          float* st = reinterpret_cast<float*>(base);
#pragma unroll
          for (int j = 0; j < 16; ++j) st[(u * 16 + j) * (lop + 1) + row] = v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) st_own_v4(X + (uint32_t)(row * hs * 4 + (((u * 4 + j) ^ (row & 7)) << 4)), *reinterpret_cast<uint4*>(v + 4 * j));
        }
      }
    operands_ready();
  }

  // four neighbours at a time; old weights of the next four are on their way while these are stored
  {
    const float* st = reinterpret_cast<const float*>(base);
    float* wts = reinterpret_cast<float*>(p.o.out);
    const int per = p.tall ? (lo * width + 3) / 4 : (width + 3) / 4, fours = p.tall ? per : per * lo;
    const bool vec_out = p.o.dtype == kOrthF32 || moving ? (reinterpret_cast<uintptr_t>(p.o.out) & 15) == 0 && ((p.tall ? lo * (int64_t)c0 | (int64_t)p.o.rows * p.o.cols : p.hi) & 3) == 0 : false;
    struct Four { int left, r, c; int64_t at; float w[4]; };
    auto fetch4 = [&](int i, Four& t) {
      t.r = p.tall ? 0 : i / per;
      t.c = (p.tall ? i : i % per) * 4;
      t.left = i < fours ? (p.tall ? lo * width : width) - t.c : 0;
      t.at = at0 + (p.tall ? (int64_t)c0 * lo : (int64_t)t.r * p.hi + c0) + t.c;
      if (!moving) return;
      if (vec_out && t.left >= 4) *reinterpret_cast<float4*>(t.w) = *reinterpret_cast<const float4*>(wts + t.at);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j) t.w[j] = j < t.left ? wts[t.at + j] : 0.f;
    };
    Four ahead[2];
    fetch4(tid, ahead[0]);
    fetch4(tid + kSmallThreads, ahead[1]);
    for (int i = tid; i < fours; i += kSmallThreads) {
      Four t = ahead[0];
      ahead[0] = ahead[1];
      fetch4(i + 2 * kSmallThreads, ahead[1]);
      float v[4];
      if (p.tall) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { const int e = t.c + j; v[j] = j < t.left ? st[e / lo * (lop + 1) + e % lo] : 0.f; }
      } else {
        *reinterpret_cast<float4*>(v) = ld_own_v4(X + (uint32_t)(t.r * hs * 4 + (((t.c >> 2) ^ (t.r & 7)) << 4)));
      }
      if (moving)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = t.w[j] - p.o.lr * v[j];
      if (vec_out && t.left >= 4) {
        *reinterpret_cast<float4*>(wts + t.at) = *reinterpret_cast<float4*>(v);
        continue;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j >= t.left) continue;
        if (moving || p.o.dtype == kOrthF32) wts[t.at + j] = v[j];
        else if (p.o.dtype == kOrthBF16) reinterpret_cast<__nv_bfloat16*>(p.o.out)[t.at + j] = __float2bfloat16_rn(v[j]);
        else reinterpret_cast<__half*>(p.o.out)[t.at + j] = __float2half_rn(v[j]);
      }
    }
  }
  if (tid == 0 && abort_flag != 0) set_status(p.o.status, kWaitTimeout, blockIdx.x, 500);
  if (p.cl > 1) cluster_sync_all();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ------------------------------------------------------------------ matrices with a short side of at most 16
// Such a matrix stays in registers: a thread holds whole columns of X (C of the longer side's), A is summed over threads, warps
// and CTAs of a cluster, and X = (a I + b A + c A²) X is C · lo² multiplications of a thread.  fp32 throughout, no tensor
// cores: a product of 16 rows would leave seven eighths of theirs idle, and their cut sums are what the last bits of so
// small a result would show.
constexpr int kThinThreads = 256, kThinColumns = 1024;     // of a CTA

struct ThinArgs {
  OrthArgs o;
  int lo, hi, tall, cl;
};

// Sums over the lanes of a warp: lane l ends up with v[0..PL) = the sums of values PL·l.. of the N (padded to 32 PL).  Halves
// are exchanged, so that it takes N shuffles instead of 5 N.
template <int PL, int kHalf = 16>
__device__ __forceinline__ void warp_scatter_sum(float (&v)[32 * PL], int lane) {
  const bool upper = lane & kHalf;
#pragma unroll
  for (int i = 0; i < kHalf * PL; ++i) {
    const float keep = upper ? v[i + kHalf * PL] : v[i], give = upper ? v[i] : v[i + kHalf * PL];
    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, kHalf);
  }
  if constexpr (kHalf > 1) warp_scatter_sum<PL, kHalf / 2>(v, lane);
}

template <int LO, int C>
__global__ void __launch_bounds__(kThinThreads, 1)
k_orth_thin(const __grid_constant__ ThinArgs p) {
  constexpr int kSums = LO * (LO + 1) / 2, PL = (kSums + 31) / 32, kWarps = kThinThreads / 32;
  __shared__ float part[kWarps][32 * PL], all[2][16][32 * PL];
  __shared__ __align__(16) float a[LO][LO], b[LO][LO < 4 ? 4 : LO];
  __shared__ double norms[kWarps], slices[16];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.cl > 1 ? (int)cluster_rank() : 0, z = blockIdx.x / p.cl;
  const int64_t at0 = (int64_t)z * p.o.rows * p.o.cols;
  const int64_t by_row = p.tall ? 1 : p.hi, by_col = p.tall ? p.lo : 1;
  pdl_wait();

  float x[C][LO];
  double acc = 0.0;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = rank * (kThinThreads * C) + k * kThinThreads + tid;
    const int64_t at = at0 + c * by_col;
    float m[LO];
#pragma unroll
    for (int r = 0; r < LO; ++r) x[k][r] = r < p.lo && c < p.hi ? load_as(p.o.x, at + r * by_row, p.o.dtype) : 0.f;
    if (p.o.m != nullptr) {
#pragma unroll
      for (int r = 0; r < LO; ++r) m[r] = r < p.lo && c < p.hi ? p.o.m[at + r * by_row] : 0.f;
#pragma unroll
      for (int r = 0; r < LO; ++r) {
        m[r] = p.o.momentum * m[r] + x[k][r];
        x[k][r] = update_direction(x[k][r], m[r], p.o.momentum, p.o.nesterov);
        if (r < p.lo && c < p.hi) p.o.m[at + r * by_row] = m[r];
      }
    }
#pragma unroll
    for (int r = 0; r < LO; ++r) acc += (double)x[k][r] * x[k][r];
  }
  acc = warp_sum_d(acc);
  if (lane == 0) norms[warp] = acc;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < kWarps; ++i) total += norms[i];
  if (p.cl > 1) {
    cluster_sync_all();                                   // every CTA runs
    if (tid < p.cl)
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_u32(smem_u32(&slices[rank]), (uint32_t)tid)), "d"(total) : "memory");
    cluster_sync_all();
    total = 0.0;
    for (int i = 0; i < p.cl; ++i) total += slices[i];
  }
  const double f = 1.0 / (sqrt(total) + (double)p.o.eps);
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int r = 0; r < LO; ++r) x[k][r] = (float)((double)x[k][r] * f);

  for (int step = 0; step < p.o.steps; ++step) {
    // A, the sums on and above the diagonal row by row
    {
      float v[32 * PL];
#pragma unroll
      for (int i = 0; i < LO; ++i)
#pragma unroll
        for (int j = i; j < LO; ++j) {
          const int n = i * LO - i * (i - 1) / 2 + j - i;
          v[n] = x[0][i] * x[0][j];
#pragma unroll
          for (int k = 1; k < C; ++k) v[n] += x[k][i] * x[k][j];
        }
#pragma unroll
      for (int n = kSums; n < 32 * PL; ++n) v[n] = 0.f;
      warp_scatter_sum<PL>(v, lane);
#pragma unroll
      for (int i = 0; i < PL; ++i) part[warp][lane * PL + i] = v[i];
    }
    __syncthreads();
    float sum = 0.f;
    if (tid < kSums)
#pragma unroll
      for (int i = 0; i < kWarps; ++i) sum += part[i][tid];
    if (p.cl > 1) {                                       // to every CTA; the steps take turns, so one barrier is enough
      if (tid < kSums)
        for (int s = 0; s < p.cl; ++s)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_u32(smem_u32(&all[step & 1][rank][tid]), (uint32_t)s)), "f"(sum) : "memory");
      cluster_sync_all();
      sum = 0.f;
      if (tid < kSums)
        for (int s = 0; s < p.cl; ++s) sum += all[step & 1][s][tid];
    }
    if (tid < kSums) {
      int i = 0, j = tid;
      while (j >= LO - i) { j -= LO - i; ++i; }
      a[i][i + j] = sum;
      a[i + j][i] = sum;
    }
    __syncthreads();
    if (tid < LO * LO) {
      const int i = tid / LO, j = tid % LO;
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < LO; ++k) sq = fmaf(a[i][k], a[k][j], sq);
      b[i][j] = fmaf(kNsC, sq, kNsB * a[i][j]) + (i == j ? kNsA : 0.f);
    }
    __syncthreads();
    float y[C][LO];
#pragma unroll
    for (int i = 0; i < LO; ++i) {
      float row[LO];
#pragma unroll
      for (int j = 0; j < LO; j += 4) {
        const float4 t = *reinterpret_cast<const float4*>(&b[i][j]);
        row[j] = t.x;
        if (j + 1 < LO) row[j + 1] = t.y;
        if (j + 2 < LO) row[j + 2] = t.z;
        if (j + 3 < LO) row[j + 3] = t.w;
      }
#pragma unroll
      for (int k = 0; k < C; ++k) {
        float t = row[0] * x[k][0];
#pragma unroll
        for (int j = 1; j < LO; ++j) t = fmaf(row[j], x[k][j], t);
        y[k][i] = t;
      }
    }
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int i = 0; i < LO; ++i) x[k][i] = y[k][i];
  }

#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = rank * (kThinThreads * C) + k * kThinThreads + tid;
    if (c >= p.hi) continue;
    const int64_t at = at0 + c * by_col;
    float* out = reinterpret_cast<float*>(p.o.out);
    float w[LO];
#pragma unroll
    for (int r = 0; r < LO; ++r) w[r] = p.o.m != nullptr && r < p.lo ? out[at + r * by_row] : 0.f;
#pragma unroll
    for (int r = 0; r < LO; ++r) {
      if (r >= p.lo) continue;
      const int64_t to = at + r * by_row;
      if (p.o.m != nullptr) out[to] = w[r] - p.o.lr * x[k][r];
      else if (p.o.dtype == kOrthF32) out[to] = x[k][r];
      else if (p.o.dtype == kOrthBF16) reinterpret_cast<__nv_bfloat16*>(p.o.out)[to] = __float2bfloat16_rn(x[k][r]);
      else reinterpret_cast<__half*>(p.o.out)[to] = __float2half_rn(x[k][r]);
    }
  }
  if (p.cl > 1) cluster_sync_all();                       // no CTA leaves while another may still write to it
}

}  // namespace psb

using namespace psb;

namespace {

struct OrthPlan {
  int lo, hi, tall;
  Tiling gram[2], square[2], step[2];         // with one plane, with two
  int64_t ldx, xplane, ldl, lplane;
  int64_t part, x0, x1, a, a2, b, slots, total;
  int thin;                                    // a cluster of cl CTAs of k_orth_thin, thin columns a thread
  int small, lop, hs, cl, a_off, a2_off, p_off, smem;      // small: a cluster of cl CTAs holds the matrix
};

constexpr int kSmallSmem = 226 * 1024;      // of 227 KB
// How many CTAs hold a matrix with a short side of at most 128: the cheapest number by this estimate of a step's cycles,
// which follows clock readings of 64x64 (5.4 k, one CTA), 128x128 (18 k, one) and 64x2048 (17.8 k on 4 CTAs).
bool small_plan(OrthPlan& p, int batch, int largest) {
  if (p.lo > 128) return false;
  p.lop = (p.lo + 15) / 16 * 16;
  const int square = 4 * p.lop * ((p.lop + 63) / 64 * 64);
  double least = 1e300;
  for (int cl = 1; cl <= largest; cl *= 2) {
    const int64_t hs = (((int64_t)p.hi + cl - 1) / cl + 63) / 64 * 64;
    if (hs > 512 || (hs + 127) / 128 * 2 * p.lop > 512) continue;                            // of TMEM
    const int sums = cl > 1 ? 4 * p.lop * p.lop : 0;
    const int bytes = 4 * p.lop * (int)hs + 2 * square + sums + (128 - p.lop) * 128;        // tiles are read as 128 rows
    if (bytes + 1024 > kSmallSmem) continue;
    const double rounds = (double)(((int64_t)batch * cl + 147) / 148), wide = p.lop > 64 ? 2.0 : 1.0;
    const double t = rounds * (wide * (4000.0 + 20.0 * (double)hs) + (cl > 1 ? 4500.0 : 0.0));
    if (t >= least) continue;
    least = t;
    p.hs = (int)hs; p.cl = cl;
    p.a_off = 4 * p.lop * p.hs; p.a2_off = p.a_off + square; p.p_off = p.a2_off + square;
    // more than half of an SM's shared memory, so that no two CTAs of a cluster meet on an SM: each takes all of its TMEM
    p.smem = bytes + 1024 < 120 * 1024 ? 120 * 1024 : bytes + 1024;
  }
  return least < 1e300;
}

bool orth_args_ok(const OrthArgs& a) {
  return a.batch > 0 && a.rows > 0 && a.cols > 0 && a.batch <= 65535 && a.rows <= (1 << 30) && a.cols <= (1 << 30) && a.steps > 0 &&
         a.dtype >= kOrthF32 && a.dtype <= kOrthF16;
}

// How many CTAs hold a matrix with a short side of at most 16, and how many columns a thread: as few columns as the SMs and the
// clusters allow, as a step's work is the columns' and its barriers cost the same.
bool thin_plan(OrthPlan& p, int batch, int largest) {
  if (p.lo > 16) return false;
  for (int c = 1; c <= kThinColumns / kThinThreads; c *= 2)
    for (int cl = 1; cl <= largest; cl *= 2)
      if ((int64_t)cl * kThinThreads * c >= p.hi && ((int64_t)batch * cl <= 148 || c == kThinColumns / kThinThreads)) {
        p.thin = c;
        p.cl = cl;
        return true;
      }
  return false;
}

// The largest cluster of k_orth_small that the current GPU takes: 16 CTAs, where its GPCs have as many SMs, 8 for certain;
// 0 where it cannot run.
int largest_cluster() {
  static int known[kMaxDevices] = {};            // one more
  int dev = 0;
  if (sm_count(&dev) <= 0) return 0;
  if (known[dev] == 0) {
    cudaError_t e = cudaFuncSetAttribute(k_orth_small, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmallSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_orth_small, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    int largest = 0;
    for (int cl = 16; cl >= 8 && e == cudaSuccess && largest == 0; cl /= 2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)cl);
      cfg.blockDim = dim3(kSmallThreads);
      cfg.dynamicSmemBytes = kSmallSmem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = (unsigned)cl; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, k_orth_small, &cfg) == cudaSuccess && clusters > 0) largest = cl;
    }
    cudaGetLastError();                          // what the question left behind
    known[dev] = largest + 1;
  }
  return known[dev] - 1;
}

struct OrthKey {
  int batch, rows, cols, largest;
  bool operator==(const OrthKey& o) const { return batch == o.batch && rows == o.rows && cols == o.cols && largest == o.largest; }
};

OrthPlan make_orth_plan(const OrthKey& a) {
  OrthPlan p = {};
  p.tall = a.rows > a.cols;
  p.lo = p.tall ? a.cols : a.rows;
  p.hi = p.tall ? a.rows : a.cols;
  // registers, shared memory, or the general way
  if ((int64_t)a.batch * 16 < (1 << 30) && thin_plan(p, a.batch, a.largest)) return p;
  if ((int64_t)a.batch * 16 < (1 << 30) && small_plan(p, a.batch, a.largest)) { p.small = 1; return p; }
  int64_t slots = 0;
  for (int k = 0; k < 2; ++k) {
    p.gram[k] = choose_tiling(a.batch, p.lo, p.lo, p.hi, k + 1, true, 32, 2);
    p.square[k] = choose_tiling(a.batch, p.lo, p.lo, p.lo, k + 1, true, 8);
    p.step[k] = choose_tiling(a.batch, a.rows, a.cols, p.lo, k + 1, false, 1);
    for (const Tiling& t : {p.gram[k], p.square[k]}) if (t.splits > 1 && t.splits > slots) slots = t.splits;
  }
  p.ldx = ((int64_t)a.cols + 7) / 8 * 8;
  p.xplane = p.ldx * a.rows;
  p.ldl = ((int64_t)p.lo + 7) / 8 * 8;
  p.lplane = p.ldl * p.lo;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  p.part = take((int64_t)a.batch * kNormBlocks * 8);
  p.x0 = take(p.xplane * 4 * a.batch);
  p.x1 = take(p.xplane * 4 * a.batch);
  p.a = take(p.lplane * 4 * a.batch);
  p.a2 = take(p.lplane * 4 * a.batch);
  p.b = take(p.lplane * 4 * a.batch);
  if (slots > 0) p.slots = take(slots * a.batch * p.lo * up4(p.lo) * 4);
  p.total = at;
  return p;
}

template <int LO, int C>
int thin_launch(Chain& chain, const ThinArgs& q) {
  int dev = 0;
  if (sm_count(&dev) <= 0) return (int)cudaErrorInvalidDevice;
  static bool attr[kMaxDevices] = {};
  if (!attr[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k_orth_thin<LO, C>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
    attr[dev] = true;
  }
  return chain.launch(k_orth_thin<LO, C>, dim3((unsigned)(q.o.batch * q.cl)), kThinThreads, 0, q.cl, q);
}
template <int LO>
int thin_rows(Chain& chain, int columns, const ThinArgs& q) {
  return columns == 1 ? thin_launch<LO, 1>(chain, q) : columns == 2 ? thin_launch<LO, 2>(chain, q) : thin_launch<LO, 4>(chain, q);
}

// a thread keeps the plans of the sizes that it met last: the search for tiles takes microseconds
OrthPlan orth_plan(const OrthArgs& a) {
  struct Entry { OrthKey key; OrthPlan plan; bool used; };
  static thread_local Entry kept[16] = {};
  const OrthKey k{a.batch, a.rows, a.cols, largest_cluster()};
  Entry& e = kept[((unsigned)k.batch * 31u + (unsigned)k.rows * 7u + (unsigned)k.cols * 13u) % 16u];
  if (!e.used || !(e.key == k)) e = Entry{k, make_orth_plan(k), true};
  return e.plan;
}

}  // namespace

extern "C" {

// bytes of workspace that the call with these arguments needs (-1: arguments out of range)
int64_t psb_orthogonal_workspace(const OrthArgs* a) { return orth_args_ok(*a) ? orth_plan(*a).total : -1; }

// Returns 0, a CUDA error, or -1 without the driver's entry point for tensor maps.
int psb_orthogonal(const OrthArgs* ap, cudaStream_t s) {
  const OrthArgs& a = *ap;
  if (!orth_args_ok(a)) return (int)cudaErrorInvalidValue;
  const OrthPlan p = orth_plan(a);
  if (p.thin) {
    Chain chain{s};
    const ThinArgs q{a, p.lo, p.hi, p.tall, p.cl};
    if (p.lo <= 1) return thin_rows<1>(chain, p.thin, q);
    if (p.lo <= 2) return thin_rows<2>(chain, p.thin, q);
    if (p.lo <= 4) return thin_rows<4>(chain, p.thin, q);
    return p.lo <= 8 ? thin_rows<8>(chain, p.thin, q) : thin_rows<16>(chain, p.thin, q);
  }
  if (p.small) {
    Chain chain{s};
    const SmallArgs q{a, p.lo, p.hi, p.tall, p.lop, p.hs, p.cl, p.a_off, p.a2_off, p.p_off};
    return chain.launch(k_orth_small, dim3((unsigned)(a.batch * p.cl)), kSmallThreads, p.smem, p.cl, q);
  }
  if (p.total > a.ws_bytes || (reinterpret_cast<uintptr_t>(a.ws) & 255)) return (int)cudaErrorInvalidValue;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.ws);
  double* part = reinterpret_cast<double*>(ws + p.part);
  uint16_t* xs[2] = {reinterpret_cast<uint16_t*>(ws + p.x0), reinterpret_cast<uint16_t*>(ws + p.x1)};
  uint16_t *ab = reinterpret_cast<uint16_t*>(ws + p.a), *a2 = reinterpret_cast<uint16_t*>(ws + p.a2), *bb = reinterpret_cast<uint16_t*>(ws + p.b);
  float* slots = reinterpret_cast<float*>(ws + p.slots);
  Chain chain{s};
  const int64_t numel = (int64_t)a.rows * a.cols;
  const int64_t per = numel % 4 == 0 ? 4096 : 1024;           // elements of a block at least
  int64_t nb = (numel + per - 1) / per;
  if (nb > kNormBlocks) nb = kNormBlocks;
  int r = chain.launch(k_orth_norm, dim3((unsigned)nb, a.batch), 256, 0, 1, a.x, a.m, numel, a.dtype, a.momentum, a.nesterov, part);
  if (r) return r;
  int64_t pb = ((int64_t)a.rows * (p.ldx / 2) + 1023) / 1024;
  if (pb > 148 * 8) pb = 148 * 8;
  r = chain.launch(k_orth_pack, dim3((unsigned)pb, a.batch), 256, 0, 1, a.x, a.m, a.rows, a.cols, a.dtype, a.momentum, a.nesterov, part, (int)nb, a.eps,
                   xs[0], p.ldx, p.xplane);
  if (r) return r;

  const bool precise = a.m != nullptr || a.dtype != kOrthBF16;
  const Operand16 A{ab, p.lo, p.lo, p.ldl, p.lplane, 2 * a.batch}, A2{a2, p.lo, p.lo, p.ldl, p.lplane, 2 * a.batch},
      B{bb, p.lo, p.lo, p.ldl, p.lplane, 2 * a.batch};
  Gemm16Args g = {};
  g.batch = a.batch; g.a_z = 2; g.b_z = 2; g.splits = 1; g.status = a.status;

  CUtensorMap map_a, map_a2, map_b;
  if ((r = make_out_map(&map_a, A, 0)) != 0 || (r = make_out_map(&map_a2, A2, 0)) != 0 || (r = make_out_map(&map_b, B, 0)) != 0) return r;

  // a symmetric product of side lo, whole or split
  auto square = [&](const Tiling& t, int planes, Gemm16Args q, const Operand16& x, const Operand16& y, EpiNs::Params e, uint16_t* out, uint16_t* out2) {
    q.M = q.N = p.lo; q.sym = t.sym; q.splits = t.splits; q.kb_split = t.kb_split;
    e.M = e.N = p.lo; e.batch = a.batch;
    if (t.splits > 1) e.slots = slots;
    int rc = product16<EpiNs>(chain, planes, t.kind, q, x, y, e);
    if (rc == 0 && t.splits > 1) {
      const unsigned nt = (unsigned)((p.lo + 31) / 32);
      rc = chain.launch(k_orth_sum, dim3(nt, nt, (unsigned)a.batch), 256, 0, 1, slots, t.splits, a.batch, p.lo, t.sym ? tiling_rows(t.kind) : 0, out, out2,
                        p.ldl, p.lplane, e.alpha, e.beta, e.alpha2, e.beta2);
    }
    return rc;
  };
  for (int k = 0; k < a.steps; ++k) {
    const int planes = precise || k + 1 < a.steps ? 2 : 1;
    const Operand16 X{xs[k & 1], a.rows, a.cols, p.ldx, p.xplane, 2 * a.batch};
    // A = X Xᵀ (or Xᵀ X), and b I + c A
    Gemm16Args gg = g;
    gg.K = p.hi; gg.a_mn = gg.b_mn = p.tall;
    EpiNs::Params ea = {};
    ea.out[0] = map_a; ea.out[1] = map_a2; ea.second = 1;
    ea.alpha = kNsInv; ea.alpha2 = kNsC * kNsInv; ea.beta2 = kNsB * kNsScale;
    if ((r = square(p.gram[planes - 1], planes, gg, X, X, ea, ab, a2)) != 0) return r;
    // B = A (b I + c A) + a I
    Gemm16Args gs = g;
    gs.K = p.lo;
    EpiNs::Params eb = {};
    eb.out[0] = map_b; eb.alpha = kNsInv; eb.beta = kNsA * kNsScale;
    if ((r = square(p.square[planes - 1], planes, gs, A, A2, eb, bb, nullptr)) != 0) return r;
    // B X (or X B)
    Gemm16Args gu = g;
    gu.M = a.rows; gu.N = a.cols; gu.K = p.lo; gu.kb_split = (p.lo + kG16K - 1) / kG16K; gu.b_mn = !p.tall;
    EpiNs::Params eu = {};
    eu.M = a.rows; eu.N = a.cols; eu.batch = a.batch; eu.alpha = kNsInv;
    if (k + 1 == a.steps) { eu.result = a.out; eu.update = a.m != nullptr; eu.dtype = a.dtype; eu.lr = a.lr; }
    else if ((r = make_out_map(&eu.out[0], Operand16{xs[(k + 1) & 1], a.rows, a.cols, p.ldx, p.xplane, 2 * a.batch}, 0)) != 0) return r;
    if ((r = product16<EpiNs>(chain, planes, p.step[planes - 1].kind, gu, p.tall ? X : B, p.tall ? B : X, eu)) != 0) return r;
  }
  return 0;
}

}  // extern "C"
