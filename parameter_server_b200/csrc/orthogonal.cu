// Orthogonalised weight updates: Newton-Schulz steps on the tensor cores (gemm16.cuh).
//
//   X = U / (|U|_F + eps);   `steps` times:  A = X Xᵀ,  X ← a X + (b A + c A²) X        on the shorter side of X
//
// with the odd polynomial of the Muon optimiser, (a, b, c) = (3.4445, −4.7750, 2.0315), which brings every singular value
// of X into about [0.7, 1.2].  For the update U = g + μ m (Nesterov) or m after m ← μ m + g, and w ← w − lr X at the end.
//
// A step is three products.  A and b A + c A² are symmetric: only the tiles on and above the diagonal are made, a tile
// above it is stored a second time, transposed.  A matrix that is taller than wide is not transposed: A = Xᵀ X reads X
// MN-major, and X (b A + c A²) reads the symmetric factor either way.  The polynomial's linear terms, the scale and the
// step of the weights are in the products' epilogues.
//
// Precision.  No entry of X, A or b A + c A² exceeds 12 in magnitude (singular values of X stay below 1.3), so all are
// kept times 2^10 in fp16, as two planes (22 bits) or one (11).  A rounding made in step k is multiplied by up to a = 3.44
// in every later step where it falls on small singular values: with one plane throughout, a matrix of a few strong
// directions over weak noise (ratio 10^2 and more) comes out 4 % off, which 16-bit results show.  One plane in the
// last two steps only leaves 0.26 % (a bf16 result is rounded to 0.17 % on average); fp32 and fp16 results take two throughout
// (8e-6 for the same matrix, 3e-7 for a random one).
#include "gemm16.cuh"

namespace psb {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr float kNsScale = 1024.f, kNsInv = 1.f / 1024.f;
constexpr int kNormBlocks = 296;

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

// Momentum, and the squares of U summed in fp64 (a gradient's entries may be anywhere in fp32's range), a block's sum each.
__global__ void __launch_bounds__(256)
k_orth_norm(const void* __restrict__ x, float* __restrict__ m, int64_t numel, int dtype, float mu, int nesterov, double* __restrict__ part) {
  const int64_t base = (int64_t)blockIdx.y * numel;
  double acc = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += (int64_t)gridDim.x * 256) {
    float u = load_as(x, base + i, dtype);
    if (m != nullptr) {
      const float mv = mu * m[base + i] + u;
      m[base + i] = mv;
      u = update_direction(u, mv, mu, nesterov);
    }
    acc += (double)u * u;
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

// U / (|U| + eps) into the planes
__global__ void __launch_bounds__(256)
k_orth_pack(const void* __restrict__ x, const float* __restrict__ m, int rows, int cols, int dtype, float mu, int nesterov,
            const double* __restrict__ part, int nparts, float eps, uint16_t* __restrict__ out, int64_t ld, int64_t plane) {
  __shared__ double sh[8];
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

// v = alpha · product + beta · C, to planes (and transposed where the tile has a mirror image), to fp32 slots of a split K,
// to the result, or as a step of the weights
struct EpiNs {
  struct Params {
    uint16_t* out;
    const uint16_t* c;         // null: no second term
    float* slots;              // not null: raw sums, [split][batch][M][N]
    void* result;              // not null: the last product
    int64_t ld, plane;         // of out and c
    int M, N, batch, write_lo, read_lo, dtype, update;
    float alpha, beta, lr;
  };
  const Params& p;
  int row, z, split;
  bool mirror;
  __device__ __forceinline__ EpiNs(const Params& p_, const Gemm16Args&, const Tile16& w, int row_, int)
      : p(p_), row(row_), z(w.z), split(w.split), mirror(w.mirror) {}
  __device__ __forceinline__ void chunk(float (&v)[32], int col) {
    if (row >= p.M || col >= p.N) return;
    const int left = p.N - col;
    if (p.slots != nullptr) {
      float* dst = p.slots + (((int64_t)split * p.batch + z) * p.M + row) * p.N + col;
#pragma unroll
      for (int j = 0; j < 32; ++j) if (j < left) dst[j] = v[j];
      return;
    }
    const int64_t at = (int64_t)z * 2 * p.plane + (int64_t)row * p.ld + col;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= p.alpha;
    if (p.c != nullptr) {
      // rows are padded to 8 elements, so whole vectors may be read wherever one element of them exists
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        if (j >= left) break;
        const uint4 h = *reinterpret_cast<const uint4*>(p.c + at + j);
        const uint4 l = p.read_lo ? *reinterpret_cast<const uint4*>(p.c + at + p.plane + j) : make_uint4(0, 0, 0, 0);
        const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hs[i])), b = __half22float2(*reinterpret_cast<const __half2*>(&ls[i]));
          v[j + 2 * i] += p.beta * (a.x + b.x);
          v[j + 2 * i + 1] += p.beta * (a.y + b.y);
        }
      }
    }
    if (p.result != nullptr) {
      const int64_t to = ((int64_t)z * p.M + row) * p.N + col;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < left) {
          const float r = v[j] * kNsInv;
          if (p.update) reinterpret_cast<float*>(p.result)[to + j] -= p.lr * r;
          else if (p.dtype == kOrthF32) reinterpret_cast<float*>(p.result)[to + j] = r;
          else if (p.dtype == kOrthBF16) reinterpret_cast<__nv_bfloat16*>(p.result)[to + j] = __float2bfloat16_rn(r);
          else reinterpret_cast<__half*>(p.result)[to + j] = __float2half_rn(r);
        }
      return;
    }
    __half h[32], l[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) split16(v[j], h[j], l[j]);
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (j >= left) break;
      *reinterpret_cast<uint4*>(p.out + at + j) = make_uint4(pack_half2(h[j], h[j + 1]), pack_half2(h[j + 2], h[j + 3]),
                                                             pack_half2(h[j + 4], h[j + 5]), pack_half2(h[j + 6], h[j + 7]));
      if (p.write_lo)
        *reinterpret_cast<uint4*>(p.out + at + p.plane + j) = make_uint4(pack_half2(l[j], l[j + 1]), pack_half2(l[j + 2], l[j + 3]),
                                                                         pack_half2(l[j + 4], l[j + 5]), pack_half2(l[j + 6], l[j + 7]));
    }
    if (mirror) {
      uint16_t* dst = p.out + (int64_t)z * 2 * p.plane + (int64_t)col * p.ld + row;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < left) {
          dst[(int64_t)j * p.ld] = __half_as_ushort(h[j]);
          if (p.write_lo) dst[(int64_t)j * p.ld + p.plane] = __half_as_ushort(l[j]);
        }
    }
  }
  __device__ __forceinline__ void end() {}
};

// the splits of A's contraction to its planes
__global__ void __launch_bounds__(256)
k_orth_sum(const float* __restrict__ slots, int splits, int batch, int n, uint16_t* __restrict__ out, int64_t ld, int64_t plane) {
  const int64_t per = (int64_t)n * n, total = per * batch;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += slots[s * total + i];
    const int64_t z = i / per, e = i - z * per, r = e / n;
    uint16_t* dst = out + z * 2 * plane + r * ld + (e - r * n);
    __half h, l;
    split16(v * kNsInv, h, l);
    dst[0] = __half_as_ushort(h);
    dst[plane] = __half_as_ushort(l);
  }
}

}  // namespace psb

using namespace psb;

namespace {

struct OrthPlan {
  int lo, hi, tall, gram_tile, sq_tile, up_tile, gram_splits;
  int64_t ldx, xplane, ldl, lplane;
  int64_t part, x0, x1, a, b, slots, total;
};

// 256x256 tiles of pairs from 48 on, 128x128 from 74 on (half of the SMs), else 128x64
int orth_tile(int64_t batch, int64_t M, int64_t N, bool sym) {
  const int64_t m2 = (M + 255) / 256, n2 = (N + 255) / 256, m1 = (M + 127) / 128, n1 = (N + 127) / 128;
  if (batch * (sym ? m2 * (m2 + 1) / 2 : m2 * n2) >= 48) return 0;
  return batch * (sym ? m1 * (m1 + 1) / 2 : m1 * n1) >= 74 ? 1 : 2;
}

bool orth_args_ok(const OrthArgs& a) {
  return a.batch > 0 && a.rows > 0 && a.cols > 0 && a.batch <= 65535 && a.rows <= (1 << 30) && a.cols <= (1 << 30) && a.steps > 0 &&
         a.dtype >= kOrthF32 && a.dtype <= kOrthF16;
}

OrthPlan orth_plan(const OrthArgs& a) {
  OrthPlan p = {};
  p.tall = a.rows > a.cols;
  p.lo = p.tall ? a.cols : a.rows;
  p.hi = p.tall ? a.rows : a.cols;
  p.gram_tile = orth_tile(a.batch, p.lo, p.lo, true);
  p.sq_tile = p.gram_tile;
  p.up_tile = orth_tile(a.batch, a.rows, a.cols, false);
  p.gram_splits = 1;
  const int64_t tiles = (int64_t)a.batch * ((p.lo + 127) / 128) * ((p.lo + 63) / 64), nkb = ((int64_t)p.hi + kG16K - 1) / kG16K;
  if (p.gram_tile == 2) {
    int64_t s = 148 / tiles;
    if (s > nkb / 8) s = nkb / 8;
    if (s > 1) { const int64_t per = (nkb + s - 1) / s; p.gram_splits = (int)((nkb + per - 1) / per); }
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
  p.b = take(p.lplane * 4 * a.batch);
  if (p.gram_splits > 1) p.slots = take((int64_t)p.gram_splits * a.batch * p.lo * p.lo * 4);
  p.total = at;
  return p;
}

template <int kPlanes, bool kAMN, bool kBMN>
int ns_product(int kind, Gemm16Args g, const Operand16& a, const Operand16& b, const EpiNs::Params& ep, cudaStream_t s) {
  if (kind == 2) g.sym = 0;                     // its tiles are not square
  if (kind == 0) return launch16<Cfg16<2, 256, kPlanes, kAMN, kBMN>, EpiNs>(g, a, b, ep, s);
  if (kind == 1) return launch16<Cfg16<1, 128, kPlanes, kAMN, kBMN>, EpiNs>(g, a, b, ep, s);
  return launch16<Cfg16<1, 64, kPlanes, kAMN, kBMN>, EpiNs>(g, a, b, ep, s);
}
template <bool kAMN, bool kBMN>
int ns_planes(int planes, int kind, const Gemm16Args& g, const Operand16& a, const Operand16& b, const EpiNs::Params& ep, cudaStream_t s) {
  return planes == 2 ? ns_product<2, kAMN, kBMN>(kind, g, a, b, ep, s) : ns_product<1, kAMN, kBMN>(kind, g, a, b, ep, s);
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
  if (p.total > a.ws_bytes || (reinterpret_cast<uintptr_t>(a.ws) & 255)) return (int)cudaErrorInvalidValue;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.ws);
  double* part = reinterpret_cast<double*>(ws + p.part);
  uint16_t* xs[2] = {reinterpret_cast<uint16_t*>(ws + p.x0), reinterpret_cast<uint16_t*>(ws + p.x1)};
  uint16_t *ab = reinterpret_cast<uint16_t*>(ws + p.a), *bb = reinterpret_cast<uint16_t*>(ws + p.b);
  float* slots = reinterpret_cast<float*>(ws + p.slots);
  const int64_t numel = (int64_t)a.rows * a.cols;
  int64_t nb = (numel + 1023) / 1024;
  if (nb > kNormBlocks) nb = kNormBlocks;
  k_orth_norm<<<dim3((unsigned)nb, a.batch), 256, 0, s>>>(a.x, a.m, numel, a.dtype, a.momentum, a.nesterov, part);
  int64_t pb = ((int64_t)a.rows * (p.ldx / 2) + 1023) / 1024;
  if (pb > 148 * 8) pb = 148 * 8;
  k_orth_pack<<<dim3((unsigned)pb, a.batch), 256, 0, s>>>(a.x, a.m, a.rows, a.cols, a.dtype, a.momentum, a.nesterov, part, (int)nb, a.eps,
                                                         xs[0], p.ldx, p.xplane);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;

  const bool precise = a.m != nullptr || a.dtype != kOrthBF16;
  const Operand16 A{ab, p.lo, p.lo, p.ldl, p.lplane, 2 * a.batch}, B{bb, p.lo, p.lo, p.ldl, p.lplane, 2 * a.batch};
  Gemm16Args g = {};
  g.batch = a.batch; g.a_z = 2; g.b_z = 2; g.splits = 1; g.status = a.status;
  for (int k = 0; k < a.steps; ++k) {
    const int planes = precise || k < a.steps - 2 ? 2 : 1, next = precise || k + 1 < a.steps - 2 ? 2 : 1;
    const bool last = k + 1 == a.steps;
    const Operand16 X{xs[k & 1], a.rows, a.cols, p.ldx, p.xplane, 2 * a.batch};
    // A = X Xᵀ (or Xᵀ X)
    Gemm16Args gg = g;
    const int nkb = (p.hi + kG16K - 1) / kG16K;
    gg.M = gg.N = p.lo; gg.K = p.hi; gg.sym = 1; gg.splits = p.gram_splits; gg.kb_split = (nkb + p.gram_splits - 1) / p.gram_splits;
    EpiNs::Params ea = {};
    ea.out = ab; ea.ld = p.ldl; ea.plane = p.lplane; ea.M = ea.N = p.lo; ea.batch = a.batch; ea.write_lo = planes == 2; ea.alpha = kNsInv;
    if (p.gram_splits > 1) ea.slots = slots;
    int r = p.tall ? ns_planes<true, true>(planes, p.gram_tile, gg, X, X, ea, s) : ns_planes<false, false>(planes, p.gram_tile, gg, X, X, ea, s);
    if (r) return r;
    if (p.gram_splits > 1) {
      const int64_t total = (int64_t)a.batch * p.lo * p.lo;
      const int64_t sb = (total + 255) / 256;
      k_orth_sum<<<(unsigned)(sb < 148 * 8 ? sb : 148 * 8), 256, 0, s>>>(slots, p.gram_splits, a.batch, p.lo, ab, p.ldl, p.lplane);
    }
    // b A + c A²
    Gemm16Args gs = g;
    gs.M = gs.N = gs.K = p.lo; gs.sym = 1; gs.kb_split = (p.lo + kG16K - 1) / kG16K;
    EpiNs::Params eb = {};
    eb.out = bb; eb.c = ab; eb.ld = p.ldl; eb.plane = p.lplane; eb.M = eb.N = p.lo; eb.batch = a.batch;
    eb.write_lo = eb.read_lo = planes == 2; eb.alpha = kNsC * kNsInv; eb.beta = kNsB;
    if ((r = ns_planes<false, false>(planes, p.sq_tile, gs, A, A, eb, s)) != 0) return r;
    // a X + (b A + c A²) X (or X (b A + c A²))
    Gemm16Args gu = g;
    gu.M = a.rows; gu.N = a.cols; gu.K = p.lo; gu.kb_split = (p.lo + kG16K - 1) / kG16K;
    EpiNs::Params eu = {};
    eu.out = xs[(k + 1) & 1]; eu.c = xs[k & 1]; eu.ld = p.ldx; eu.plane = p.xplane; eu.M = a.rows; eu.N = a.cols; eu.batch = a.batch;
    eu.read_lo = planes == 2; eu.write_lo = next == 2; eu.alpha = kNsInv; eu.beta = kNsA;
    if (last) { eu.result = a.out; eu.update = a.m != nullptr; eu.dtype = a.dtype; eu.lr = a.lr; }
    r = p.tall ? ns_planes<false, false>(planes, p.up_tile, gu, X, B, eu, s) : ns_planes<false, true>(planes, p.up_tile, gu, B, X, eu, s);
    if (r) return r;
  }
  return (int)cudaGetLastError();
}

}  // extern "C"
