// Softmax cross entropy of rows over many classes, with its gradients, without keeping the scores.
//
//   s_ij = x_i · w_j        loss_i = c_i (log Σ_j e^{s_ij} − s_{i,y_i})        x [n, d], w [V, d], y_i in 0..V-1 or -1
//   G_ij = c_i (e^{s_ij − lse_i} − [j = y_i])        gx = G w        gw = Gᵀ x
//
// The scores are tiles of a product on the tensor cores (gemm16.cuh) and never leave the SM: its epilogue keeps each row's
// maximum m and sum Σ e^{s−m} over a part of a tile's classes (32 to 128), and the score of the row's label.  A second
// kernel joins the parts of a row to its log-sum-exp.
//
// For the gradients the epilogue also writes e^{s−m} · 2^15 in fp16 (relative to the part's own maximum, which is all that
// is known then), for as many classes as the workspace holds; the second kernel turns it into G in place, with one
// factor a part.  Making the scores once costs 6nVd operations instead of 8nVd, for a pass over 2 bytes an element
// (8192 rows, 131,072 classes, 2048 wide: 3.2 ms less for 0.85).  Classes beyond the workspace come in pieces, whose scores
// are made again.  gw of a piece is complete, gx is summed over the pieces in fp32.  Sums have a fixed order: results do not
// vary from run to run.
//
// Bound by the tensor cores: bf16 scores of 4096 rows against 131,072 classes, 1024 wide, take 785 us, 0.83 of the rate of a plain
// cuBLAS product; 8192 x 131,072 x 2048 with gradients takes 10.4 ms where the products alone, at its sustained rate, take 9.5.
//
// Scores, maxima, sums and losses are fp32 (in units of log2 e: 2^x is the hardware's exponential).  The exponentials keep 11
// bits (two planes for fp32: 22); the label's entry of G, where they would cancel, is made from the label's score in fp32.
// G is rounded to the operands' type: bf16 for bf16; fp16 for fp16, scaled by a power of two so that the largest
// coefficient is near 2^13; two planes of fp16 for fp32, where x and w are such planes too.
#include "gemm16.cuh"

namespace psb {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kExpScale = 15;                 // exponentials relative to their maximum are kept times 2^15

enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// Exponents of the operands' scales: x and w are multiplied by 2^x and 2^w, G by 2^g.
struct Scales { int x, w, g; };
// They are 0 for 16-bit operands and g is known where there are no coefficients; else the device finds them.
struct ScaleRef {
  Scales fixed;
  const Scales* found;         // null: as fixed
  __device__ __forceinline__ Scales get() const { return found != nullptr ? *found : fixed; }
};
// exponent that brings the magnitude with these bits into [2^top, 2^(top+1)); subnormals count as 2^-127, as the scale only
// has to be representable
__device__ __forceinline__ int scale_exp(uint32_t bits, int top) {
  if (bits == 0) return 0;
  const int k = top - ((int)(bits >> 23) - 127);
  return k > 126 ? 126 : k;
}
__device__ __forceinline__ float pow2i(int e) {       // 2^e, kept finite; 0 below the normal numbers
  e = e > 127 ? 127 : e;
  return e < -126 ? 0.f : __int_as_float((e + 127) << 23);
}
__device__ __forceinline__ float score_scale(const ScaleRef& r) { const Scales k = r.get(); return kLog2e * pow2i(-(k.x + k.w)); }
// 2^e in two factors of the same direction: the power may lie outside fp32 where what it scales does not leave it
struct Pow2 {
  float a, b;
  __device__ __forceinline__ explicit Pow2(int e) : a(pow2i(e / 2)), b(pow2i(e - e / 2)) {}
  __device__ __forceinline__ float operator*(float v) const { return v * a * b; }
};
__device__ __forceinline__ Pow2 grad_scale(const ScaleRef& r, int with_w) { const Scales k = r.get(); return Pow2(-(k.g + (with_w ? k.w : k.x))); }
__device__ __forceinline__ bool has_class(int64_t y, int V) { return y >= 0 && y < V; }

// ------------------------------------------------------------------ preparation
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v) {       // of 256 threads, in all of them
  __shared__ uint32_t sh[8];
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[threadIdx.x & 7];
  return __reduce_max_sync(0xffffffffu, v);
}
__device__ __forceinline__ uint32_t coef_max(const float* coef, const int64_t* y, int n, int V) {
  if (coef == nullptr) return __float_as_uint(1.f);
  uint32_t top = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 256) {
    const float c = coef[i];
    if (has_class(y[i], V)) top = max(top, finite_bits(c));
  }
  return block_max_u32(top);
}
// fp16 with coefficients: the scale of G alone (one block)
__global__ void __launch_bounds__(256)
k_loss_coef(const float* __restrict__ coef, const int64_t* __restrict__ y, int n, int V, Scales* out) {
  pdl_wait();
  const uint32_t top = coef_max(coef, y, n, V);
  if (threadIdx.x == 0) *out = Scales{0, 0, scale_exp(top, 13)};
}

// the largest finite magnitude that a thread finds, taking each step-th four columns from the first on (y null: all rows count)
__device__ __forceinline__ uint32_t thread_absmax(const float* a, int64_t ld, int64_t rows, int cols, const int64_t* y, int V, int64_t first,
                                                  int64_t step) {
  uint32_t top = 0;
  if (y == nullptr && ld == cols && (reinterpret_cast<uintptr_t>(a) & 15) == 0) {       // one long row, whatever its pieces' alignment
    const int64_t n = rows * cols;
#pragma unroll 4
    for (int64_t i = first; i < n / 4; i += step) {
      const float4 v = reinterpret_cast<const float4*>(a)[i];
      top = max(max(top, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
    }
    for (int64_t i = n / 4 * 4 + first; i < n; i += step) top = max(top, finite_bits(a[i]));
    return top;
  }
  const bool vec = ((reinterpret_cast<uintptr_t>(a) & 15) | (ld & 3)) == 0;
  const int per = (cols + 3) / 4;
  const int64_t total = rows * per;
  for (int64_t i = first; i < total; i += step) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 4;
    if (y != nullptr && !has_class(y[r], V)) continue;
    const float* p = a + r * ld + c;
    if (vec && c + 4 <= cols) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      top = max(max(top, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
    } else {
      for (int j = 0; j < 4 && c + j < cols; ++j) top = max(top, finite_bits(p[j]));
    }
  }
  return top;
}
// Largest finite magnitudes of fp32 operands, a block's each: blocks 0..bx-1 take x (rows without a class do not count),
// the others w.
__global__ void __launch_bounds__(256)
k_loss_absmax(const float* __restrict__ x, int64_t ldx, const float* __restrict__ w, int64_t ldw, int n, int V, int d,
              const int64_t* __restrict__ y, int bx, uint32_t* __restrict__ out) {
  pdl_wait();
  const int b = (int)blockIdx.x;
  const uint32_t top = block_max_u32(b < bx ? thread_absmax(x, ldx, n, d, y, V, (int64_t)b * 256 + threadIdx.x, (int64_t)bx * 256)
                                            : thread_absmax(w, ldw, V, d, nullptr, V, (int64_t)(b - bx) * 256 + threadIdx.x,
                                                            (int64_t)(gridDim.x - bx) * 256));
  if (threadIdx.x == 0) out[b] = top;
}

struct PackArgs {
  const void* a;               // rows of `cols` elements, any stride and alignment
  int64_t rows, ld;
  uint16_t* out;               // operand planes [plane][row][ldo]
  int64_t ldo, plane;
};
// Operands into planes of their own: blocks 0..bx-1 pack x, the others w (either may have no blocks).  Rows of x without a
// class become zeros, whatever they held.  fp32: the scales come from the blocks' maxima and are written for those who follow.
template <typename T>
__global__ void __launch_bounds__(256)
k_loss_pack(PackArgs px, PackArgs pw, int cols, const int64_t* __restrict__ y, int n, int V, const float* __restrict__ coef, int bx,
            const uint32_t* maxima, int mx, int mw, Scales* found) {
  pdl_wait();
  const bool is_x = (int)blockIdx.x < bx;
  const PackArgs& p = is_x ? px : pw;
  const int64_t nb = is_x ? bx : gridDim.x - bx, b = is_x ? blockIdx.x : blockIdx.x - bx;
  float s = 1.f;
  if (sizeof(T) == 4) {
    uint32_t tx = 0, tw = 0;
    const bool last = blockIdx.x == gridDim.x - 1;
    if (maxima == nullptr) {                 // small operands: every block looks through them itself
      if (is_x || last) tx = thread_absmax(reinterpret_cast<const float*>(px.a), px.ld, px.rows, cols, y, V, threadIdx.x, 256);
      if (!is_x) tw = thread_absmax(reinterpret_cast<const float*>(pw.a), pw.ld, pw.rows, cols, nullptr, V, threadIdx.x, 256);
    } else {
      if (is_x || last) for (int i = threadIdx.x; i < mx; i += 256) tx = max(tx, maxima[i]);
      if (!is_x) for (int i = threadIdx.x; i < mw; i += 256) tw = max(tw, maxima[mx + i]);
    }
    const int kx = scale_exp(block_max_u32(tx), 14), kw = scale_exp(block_max_u32(tw), 14);
    s = pow2i(is_x ? kx : kw);
    if (last) {
      const uint32_t tc = coef_max(coef, y, n, V);
      if (threadIdx.x == 0) *found = Scales{kx, kw, scale_exp(tc, 13)};
    }
  }
  const T* a = reinterpret_cast<const T*>(p.a);
  if (((reinterpret_cast<uintptr_t>(a) & 15) | ((p.ld * sizeof(T)) & 15)) != 0) {
    // rows of any alignment: a warp a row, two columns a thread, so that loads and stores are pieces of one row
    const int64_t warps = nb * 8;
    for (int64_t r = b * 8 + (threadIdx.x >> 5); r < p.rows; r += warps) {
      const T* src = a + r * p.ld;
      uint16_t* dst = p.out + r * p.ldo;
      const bool none = is_x && !has_class(y[r], V);
#pragma unroll 4
      for (int c = (threadIdx.x & 31) * 2; c < (int)p.ldo; c += 64) {
        const T u = !none && c < cols ? src[c] : T(0), v = !none && c + 1 < cols ? src[c + 1] : T(0);
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<uint32_t*>(dst + c) = pair16<kFmtPlanes>((float)u * s, (float)v * s, false);
          *reinterpret_cast<uint32_t*>(dst + p.plane + c) = pair16<kFmtPlanes>((float)u * s, (float)v * s, true);
        } else {
          *reinterpret_cast<uint32_t*>(dst + c) = (uint32_t)*reinterpret_cast<const uint16_t*>(&u) | (uint32_t)*reinterpret_cast<const uint16_t*>(&v) << 16;
        }
      }
    }
    return;
  }
  const int per = (int)(p.ldo / 8);
  const int64_t total = p.rows * per;
  for (int64_t i = b * 256 + threadIdx.x; i < total; i += nb * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    const T* src = a + r * p.ld + c;
    alignas(16) T v[8];
    if (is_x && !has_class(y[r], V)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = T(0);
    } else if (c + 8 <= cols) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(v)[j] = reinterpret_cast<const uint4*>(src)[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? src[j] : T(0);
    }
    uint16_t* dst = p.out + r * p.ldo + c;
    if constexpr (sizeof(T) == 4) {
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = pair16<kFmtPlanes>((float)v[2 * j] * s, (float)v[2 * j + 1] * s, false);
        l[j] = pair16<kFmtPlanes>((float)v[2 * j] * s, (float)v[2 * j + 1] * s, true);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(dst + p.plane) = make_uint4(l[0], l[1], l[2], l[3]);
    } else {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(v);
    }
  }
}

// ------------------------------------------------------------------ epilogues
// Each row's maximum and Σ 2^(s−m) over a part of a tile's classes, the score of its label, in units of log2 e, and the
// exponentials that are kept.
struct EpiScore {
  struct Params {
    CUtensorMap e;             // exponentials [plane][n][keep]
    float2* part;              // [n][per_tile · class tiles]
    float* target;             // [n]
    const int64_t* y;
    ScaleRef scale;
    int n, V, parts, per_tile, keep;
  };
  template <int kPart>
  static __device__ __forceinline__ void ahead(const Params&, const Tile16&, int, int, int) {}
  template <int kPlanes, int kPart, class Stage, class Sums, class Done>
  static __device__ __forceinline__ void run(const Params& p, const Gemm16Args&, const Tile16& w, int row0, int col0, int part, Stage& st,
                                             const Sums& sums, Done done) {
    const float scale = score_scale(p.scale);
    const int row = row0 + st.lane;
    int64_t lab = -1;
    if (row < p.n) lab = p.y[row];
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kPart; c += 32) {
      float v[32];
      sums.load(c, v);
      const int left = p.V - (col0 + c);
      if (left >= 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = j < left ? fmaxf(top, v[j]) : top;
      }
    }
    // without a finite score the reference is 0: 2^(-inf) is 0 and nothing is subtracted from an infinity
    const float m = __fmul_rn(top, scale), ref = top == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll 1
    for (int c = 0; c < kPart; c += 32) {
      float v[32];
      sums.load(c, v);
      if (c + 32 >= kPart) done();
      const int col = col0 + c, left = p.V - col;
      if (left <= 0) continue;
      if (lab >= col && lab < col + 32 && lab < p.V) {
        const int at = (int)(lab - col);
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) t = j == at ? v[j] : t;
        p.target[row] = __fmul_rn(t, scale);
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        // product and difference rounded apart, as those of the maximum and of the label are: a row whose class is certain has
        // a loss of 0, not of a rounding
        v[j] = ex2(__fsub_rn(__fmul_rn(v[j], scale), ref));
        if (left < 32) v[j] = j < left ? v[j] : 0.f;
        s += v[j];
        v[j] *= (float)(1 << kExpScale);
      }
      if (col < p.keep) st.template store<kPlanes == 2 ? kFmtPlanes : kFmtF16>(&p.e, v, row0, col, 0, false);
    }
    if (row < p.n) p.part[(int64_t)row * p.parts + w.tn * p.per_tile + part] = make_float2(top == -INFINITY ? top : m, s);
  }
};

// G of a piece of the classes, in the operands' type, from scores made again
struct EpiG {
  struct Params {
    CUtensorMap g;             // [plane][n][len]
    const float* lse;          // [n], log2
    const float* coef;
    const int64_t* y;
    ScaleRef scale;
    int n, V, len, v0, dtype;
  };
  template <int kPart>
  static __device__ __forceinline__ void ahead(const Params&, const Tile16&, int, int, int) {}
  template <int kPlanes, int kPart, class Stage, class Sums, class Done>
  static __device__ __forceinline__ void run(const Params& p, const Gemm16Args&, const Tile16&, int row0, int col0, int, Stage& st,
                                             const Sums& sums, Done done) {
    const float scale = score_scale(p.scale);
    const int row = row0 + st.lane;
    float c = 0.f, lse = 0.f;
    int64_t lab = -1;
    if (row < p.n && has_class(p.y[row], p.V)) {
      lab = p.y[row] - p.v0;
      c = (p.coef != nullptr ? p.coef[row] : 1.f) * pow2i(p.scale.get().g);
      lse = p.lse[row];
    }
    const bool none = row >= p.n || !has_class(p.y[row], p.V);
#pragma unroll 1
    for (int k = 0; k < kPart; k += 32) {
      float v[32];
      sums.load(k, v);
      if (k + 32 >= kPart) done();
      const int col = col0 + k;
      if (col >= p.len) continue;
      const int at = lab >= col && lab < col + 32 ? (int)(lab - col) : -1;
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = none ? 0.f : c * (ex2(fmaf(v[j], scale, -lse)) - (at == j ? 1.f : 0.f));
      if constexpr (kPlanes == 2) st.template store<kFmtPlanes>(&p.g, v, row0, col, 0, false);
      else if (p.dtype == kBF16) st.template store<kFmtBF16>(&p.g, v, row0, col, 0, false);
      else st.template store<kFmtF16>(&p.g, v, row0, col, 0, false);
    }
  }
};

__device__ __forceinline__ void store_as(void* out, int64_t at, float v, int dtype) {
  if (dtype == kF32) reinterpret_cast<float*>(out)[at] = v;
  else if (dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
}

// A gradient: to the result, or as fp32 sums to `acc` (piece by piece, or one slot per split of K)
struct EpiGrad {
  struct Params {
    CUtensorMap map;           // of the result, where it is 16-bit and aligned
    void* out;
    float* acc;
    int64_t slot;
    ScaleRef scale;
    int M, N, dtype, with_w, by_map;
    int read, write;           // acc is added to the product; the sum goes to acc instead of the result
  };
  template <int kPart>
  static __device__ __forceinline__ void ahead(const Params& p, const Tile16& w, int row, int col, int lane) {
    if (p.read && row + lane < p.M) prefetch_l2<kPart>(p.acc + w.split * p.slot + (int64_t)(row + lane) * p.N, col, p.N);
  }
  template <int kPlanes, int kPart, class Stage, class Sums, class Done>
  static __device__ __forceinline__ void run(const Params& p, const Gemm16Args&, const Tile16& w, int row0, int col0, int, Stage& st,
                                             const Sums& sums, Done done) {
    const Pow2 scale = grad_scale(p.scale, p.with_w);
#pragma unroll 1
    for (int k = 0; k < kPart; k += 32) {
      float v[32];
      sums.load(k, v);
      if (k + 32 >= kPart) done();
      const int col = col0 + k;
      if (row0 >= p.M || col >= p.N) continue;
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = scale * v[j];
      if (kPlanes == 1 && p.by_map) {
        if (p.dtype == kBF16) st.template store<kFmtBF16>(&p.map, v, row0, col, 0, false);
        else st.template store<kFmtF16>(&p.map, v, row0, col, 0, false);
        continue;
      }
      const int rows = p.M - row0 < 32 ? p.M - row0 : 32, mine = col + st.lane;
      const bool in = mine < p.N;
      const int64_t at = (int64_t)row0 * p.N + mine;
      float* acc = p.acc != nullptr ? p.acc + w.split * p.slot + at : nullptr;
      st.by_rows(v, [&](auto value) {
        if (!in) return;
        if (!p.read) {                                       // by type and by pointer: an index for each row was half of this loop
          if (p.write || p.dtype == kF32) {
            float* dst = p.write ? acc : reinterpret_cast<float*>(p.out) + at;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, dst += p.N) *dst = value(r);
          } else if (p.dtype == kBF16) {
            __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, dst += p.N) *dst = __float2bfloat16_rn(value(r));
          } else {
            __half* dst = reinterpret_cast<__half*>(p.out) + at;
#pragma unroll 8
            for (int r = 0; r < rows; ++r, dst += p.N) *dst = __float2half_rn(value(r));
          }
          return;
        }
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += 16) {
          float t[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) t[i] = in && r0 + i < rows ? acc[(int64_t)(r0 + i) * p.N] : 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            t[i] += value(r0 + i);
            if (!in || r0 + i >= rows) continue;
            if (p.write) acc[(int64_t)(r0 + i) * p.N] = t[i];
            else store_as(p.out, at + (int64_t)(r0 + i) * p.N, t[i], p.dtype);
          }
        }
      });
    }
  }
};

// ------------------------------------------------------------------ joining
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x), ref = m == -INFINITY ? 0.f : m;
  return make_float2(m, a.y * ex2(a.x - ref) + b.y * ex2(b.x - ref));
}
// the parts of a row, joined by kLanes threads of a block (a warp, or the block of 256), in all of them
template <int kLanes>
__device__ __forceinline__ float2 join_row(const float2* part, int parts, int ln) {
  float2 a = make_float2(-INFINITY, 0.f);
  for (int q = ln; q < parts; q += kLanes) a = join(a, part[q]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = join(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, o), __shfl_xor_sync(0xffffffffu, a.y, o)));
  if (kLanes > 32) {
    __shared__ float2 sh[8];
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
    __syncthreads();
    a = sh[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) a = join(a, sh[i]);
  }
  return a;
}

struct JoinArgs {
  const float2* part;
  const float* target;
  const int64_t* y;
  const float* coef;
  float* lse;
  float* loss;
  uint16_t* g;                 // exponentials that become G; null: the losses alone
  int64_t ldg, plane;
  const uint16_t* x;           // rows that are copied with zeros where there is no class; null: packed already
  uint16_t* x_out;
  int64_t ldx, ldxo;
  ScaleRef scale;
  int n, V, d, parts, shift, keep, dtype;    // 2^shift: classes of a part
  uint32_t* status;
};
// A row's log-sum-exp (log2) and loss and, in place, its kept exponentials to G.  kLanes threads a row; blockIdx.y shares
// the classes of a row where there are few rows.  Bound by reading and writing G.
template <int kLanes>
__global__ void __launch_bounds__(256)
k_loss_rows(const __grid_constant__ JoinArgs p) {
  pdl_wait();
  const int ln = threadIdx.x % kLanes, row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (kLanes == 32 && row >= p.n) return;
  const float2* part = p.part + (int64_t)row * p.parts;
  const float2 a = join_row<kLanes>(part, p.parts, ln);
  const float l2 = log2f(a.y), lse = a.x + l2;
  const int64_t lab = p.y[row];
  const bool ok = has_class(lab, p.V);
  const float c = ok ? (p.coef != nullptr ? p.coef[row] : 1.f) : 0.f;
  const float target = ok ? p.target[row] : 0.f;
  if (ln == 0 && blockIdx.y == 0) {
    if (lab != -1 && !ok) set_status(p.status, kBadIndex, (uint32_t)row, (uint32_t)lab);
    p.lse[row] = lse;
    p.loss[row] = ok ? c * (kLn2 * ((a.x - target) + l2)) : 0.f;
  }
  if (p.g == nullptr) return;
  if (p.x != nullptr && blockIdx.y == 0) {
    // 16-byte aligned rows of any length: what lies between the end of a row and its stride is never read by a product
    for (int i = ln * 8; i < p.d; i += kLanes * 8) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (ok) {
        if (i + 8 <= p.d) {
          v = *reinterpret_cast<const uint4*>(p.x + row * p.ldx + i);
        } else {
          uint16_t t[8] = {};
#pragma unroll
          for (int j = 0; j < 8; ++j) if (i + j < p.d) t[j] = p.x[row * p.ldx + i + j];
          v = make_uint4(t[0] | t[1] << 16, t[2] | t[3] << 16, t[4] | t[5] << 16, t[6] | t[7] << 16);
        }
      }
      *reinterpret_cast<uint4*>(p.x_out + row * p.ldxo + i) = v;
    }
  }
  const int kg = p.scale.get().g;
  const float cg = c * pow2i(kg), at_label = cg * (ex2((target - a.x) - l2) - 1.f);
  const float shift = (float)kExpScale + l2;
  uint16_t* g = p.g + (int64_t)row * p.ldg;
  // four eights a thread at a time: their loads do not wait for one another
  const int step = gridDim.y * kLanes * 8;
  for (int first = (blockIdx.y * kLanes + ln) * 8; first < p.keep; first += 4 * step) {
    uint4 h[4], l[4];
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int col = first + k * step;
      if (col >= p.keep) break;
      h[k] = *reinterpret_cast<const uint4*>(g + col);
      if (p.dtype == kF32) l[k] = *reinterpret_cast<const uint4*>(g + p.plane + col);
      f[k] = part[col >> p.shift].x;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int col = first + k * step;
      if (col >= p.keep) break;
      const float scale = cg * ex2((f[k] - a.x) - shift);
      const int at = lab >= col && lab < col + 8 ? (int)(lab - col) : -1;
      uint32_t hs[4] = {h[k].x, h[k].y, h[k].z, h[k].w}, ls[4] = {l[k].x, l[k].y, l[k].z, l[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hs[i]));
        if (p.dtype == kF32) {
          const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&ls[i]));
          v.x += u.x; v.y += u.y;
        }
        v.x = ok ? (at == 2 * i ? at_label : v.x * scale) : 0.f;
        v.y = ok ? (at == 2 * i + 1 ? at_label : v.y * scale) : 0.f;
        if (p.dtype == kBF16) {
          hs[i] = pair16<kFmtBF16>(v.x, v.y, false);
        } else {
          hs[i] = pair16<kFmtPlanes>(v.x, v.y, false);
          if (p.dtype == kF32) ls[i] = pair16<kFmtPlanes>(v.x, v.y, true);
        }
      }
      *reinterpret_cast<uint4*>(g + col) = make_uint4(hs[0], hs[1], hs[2], hs[3]);
      if (p.dtype == kF32) *reinterpret_cast<uint4*>(g + p.plane + col) = make_uint4(ls[0], ls[1], ls[2], ls[3]);
    }
  }
}

// the splits of K to the result
__global__ void __launch_bounds__(256)
k_loss_sum(const float* acc, int splits, int64_t slot, int64_t numel, void* out, int dtype) {
  pdl_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int q = 0; q < splits; ++q) v += acc[q * slot + i];
    store_as(out, i, v, dtype);
  }
}

// arguments of a call, laid out as the binding has them
struct LossArgs {
  const void* x;
  const void* w;
  const int64_t* y;
  const float* coef;
  float* loss;
  void* gx;
  void* gw;
  int64_t ldx, ldw;
  int n, V, d, dtype, want_grad, keep_mb;     // keep_mb: megabytes of exponentials that are kept
  void* ws;
  int64_t ws_bytes;
  uint32_t* status;
};

// ------------------------------------------------------------------ small calls
// Rows and classes that fit into shared memory take one launch without a workspace, in fp32 on the CUDA cores: each of the four
// launches of the general way costs 3 us of host time and 4 on the GPU, whatever its size.  One CTA, or a cluster of 8 in which each
// holds all of x, w and the scores and makes a share of the scores, which it sends to the others, and of the gradients.
//   calls behind one another with gradients, general way -> this one (on the GPU alone), us:
//     16 x 100 x 64 fp32 25 -> 16 (15 -> 9.5), bf16 23 -> 16 (10 -> 9.5); 64 x 64 x 64 (2^18) 25 -> 18 (16 -> 14);
//     1 x 500 x 64 25 -> 16.5 (19 -> 14.6); 128 x 128 x 64 (2^20) 25 -> 28 (19 -> 27), which is beyond the limit.
//   One CTA instead of 8: 16 x 100 x 64 12.9 us on the GPU, 3 x 7 x 8 the same 5.2.
// Bound by latency: loads from L2, two cluster barriers, chains of shared-memory reads.
//
// A thread makes four results next to one another, from four rows of one factor (read by all lanes alike) and a column of the
// other; where there are fewer of those than threads, neighbouring lanes share a sum.  Rows of x and w are an odd number of
// 16 bytes apart, free of bank conflicts.
struct TinyArgs {
  LossArgs a;
  int ld, ldg, cl;             // floats from a row of x and w to the next, and of the scores; CTAs of the cluster
};
constexpr int kTinyThreads = 512, kTinySmem = 200 * 1024, kTinyCtas = 8;
constexpr int kTinyRows = 512;                             // and classes
constexpr int64_t kTinyWork = 1 << 18, kTinyAlone = 1 << 12;        // rows x classes x columns: of a call, of a single CTA

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// A CTA's share of `units` results of four: sum(unit, part, parts, v) adds a part of the terms, store(unit, v) takes the sums
template <class Sum, class Store>
__device__ __forceinline__ void four_at_once(int units, int terms, int rank, int cl, Sum sum, Store store) {
  const int per = (units + cl - 1) / cl, first = rank * per, left = units - first, count = left < per ? left : per;
  int shift = 0;
  while (shift < 5 && per << (shift + 1) <= kTinyThreads && terms >> (shift + 1) >= 4) ++shift;
  const int lane = threadIdx.x & 31;
  for (int b = threadIdx.x; b - lane < count << shift; b += kTinyThreads) {
    const int u = b >> shift, part = b & ((1 << shift) - 1);
    float v[4] = {};
    if (u < count) sum(first + u, part, 1 << shift, v);
    for (int o = 1; o < 1 << shift; o <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (u < count && part == 0) store(first + u, v);
  }
}

template <typename T>
__global__ void __launch_bounds__(kTinyThreads, 1)
k_loss_tiny(const __grid_constant__ TinyArgs q) {
  extern __shared__ __align__(16) float tiny_smem[];
  const LossArgs& a = q.a;
  const int n = a.n, V = a.V, d = a.d, ld = q.ld, ldg = q.ldg, n4 = (n + 3) / 4 * 4, v4 = (V + 3) / 4 * 4;
  float *xs = tiny_smem, *wsm = xs + n4 * ld, *S = wsm + v4 * ld;
  const int tid = threadIdx.x, lane = tid & 31, rank = q.cl > 1 ? (int)cluster_rank() : 0;

  // fours of columns; zeros beside the matrices and in rows without a class
  const int per_row = ld / 4, fours = (n4 + v4) * per_row;
#pragma unroll 4
  for (int i = tid; i < fours; i += kTinyThreads) {
    const int r = i / per_row, c = (i - r * per_row) * 4, j = r - n4;
    const bool in = r < n4 ? r < n && has_class(a.y[r < n ? r : 0], V) : j < V;
    const T* src = r < n4 ? reinterpret_cast<const T*>(a.x) + (int64_t)r * a.ldx : reinterpret_cast<const T*>(a.w) + (int64_t)j * a.ldw;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = in && c + k < d ? as_float(src[c + k]) : 0.f;
    *reinterpret_cast<float4*>(xs + r * ld + c) = make_float4(v[0], v[1], v[2], v[3]);
  }
  if (q.cl > 1) cluster_sync_all();                       // every CTA runs
  else __syncthreads();

  // scores in units of log2 e: four rows against a class
  four_at_once(n4 / 4 * V, ld / 4, rank, q.cl,
    [&](int u, int part, int parts, float (&v)[4]) {
      const int i = u / V, j = u - i * V;
      const float4 *wr = reinterpret_cast<const float4*>(wsm + j * ld), *xr = reinterpret_cast<const float4*>(xs + i * 4 * ld);
      for (int k0 = part; k0 < per_row; k0 += 16 * parts) {
        float t[4] = {};
#pragma unroll 4
        for (int k = k0; k < per_row && k < k0 + 16 * parts; k += parts) {
          const float4 w = wr[k];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 x = xr[r * per_row + k];
            t[r] = fmaf(x.x, w.x, fmaf(x.y, w.y, fmaf(x.z, w.z, fmaf(x.w, w.w, t[r]))));
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += t[r];
      }
    },
    [&](int u, const float (&v)[4]) {
      const int i = u / V, j = u - i * V;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float* at = S + (i * 4 + r) * ldg + j;
        const float s = __fmul_rn(v[r], kLog2e);
        if (q.cl == 1) *at = s;
        else
          for (int c = 0; c < q.cl; ++c)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_u32(smem_u32(at), (uint32_t)c)), "f"(s) : "memory");
      }
    });
  if (q.cl > 1) cluster_sync_all();
  else __syncthreads();

  // losses, and the gradient of the scores in place: a few lanes a row
  int shift = 0;
  while (shift < 5 && 4 << shift < V) ++shift;
  for (int b = tid; b - lane < n << shift; b += kTinyThreads) {
    const int row = b >> shift, part = b & ((1 << shift) - 1), parts = 1 << shift;
    const bool in = row < n;
    float* s = S + (in ? row : 0) * ldg;
    float top = -INFINITY, sum = 0.f;
    if (in) for (int j = part; j < V; j += parts) top = fmaxf(top, s[j]);
    for (int o = 1; o < parts; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.f : top;
    if (in) for (int j = part; j < V; j += parts) sum += ex2(s[j] - ref);
    for (int o = 1; o < parts; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!in) continue;
    const float l2 = log2f(sum);
    const int64_t lab = a.y[row];
    const bool ok = has_class(lab, V);
    const float c = ok ? (a.coef != nullptr ? a.coef[row] : 1.f) : 0.f;
    if (part == 0 && rank == 0) {
      if (lab != -1 && !ok) set_status(a.status, kBadIndex, (uint32_t)row, (uint32_t)lab);
      if (!ok) a.loss[row] = 0.f;
    }
    if (ok && (int)lab % parts == part && rank == 0) a.loss[row] = c * (kLn2 * ((top - s[lab]) + l2));
    if (!a.want_grad) continue;
    for (int j = part; j < ldg; j += parts) {
      const float p = ok && j < V ? ex2((s[j] - top) - l2) : 0.f;
      s[j] = ok && j < V ? c * (j == lab ? p - 1.f : p) : 0.f;
    }
  }
  if (!a.want_grad) return;
  __syncthreads();

  if (a.gx != nullptr)
    four_at_once(n4 / 4 * d, ldg / 4, rank, q.cl,           // four rows, a column
      [&](int u, int part, int parts, float (&v)[4]) {
        const int i = u / d, c = u - i * d, terms = ldg / 4;
        const float4* g = reinterpret_cast<const float4*>(S + i * 4 * ldg);
        for (int k0 = part; k0 < terms; k0 += 16 * parts) {
          float t[4] = {};
#pragma unroll 4
          for (int k = k0; k < terms && k < k0 + 16 * parts; k += parts) {
            const float* w = wsm + k * 4 * ld + c;
            const float w0 = w[0], w1 = w[ld], w2 = w[2 * ld], w3 = w[3 * ld];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float4 x = g[r * terms + k];
              t[r] = fmaf(x.x, w0, fmaf(x.y, w1, fmaf(x.z, w2, fmaf(x.w, w3, t[r]))));
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += t[r];
        }
      },
      [&](int u, const float (&v)[4]) {
        const int i = u / d, c = u - i * d;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i * 4 + r < n) store_as(a.gx, (int64_t)(i * 4 + r) * d + c, v[r], a.dtype);
      });
  four_at_once(v4 / 4 * d, n, rank, q.cl,                   // four classes, a column
    [&](int u, int part, int parts, float (&v)[4]) {
      const int j = u / d, c = u - j * d;
      for (int k0 = part; k0 < n; k0 += 64 * parts) {
        float t[4] = {};
#pragma unroll 4
        for (int k = k0; k < n && k < k0 + 64 * parts; k += parts) {
          const float4 g = *reinterpret_cast<const float4*>(S + k * ldg + j * 4);
          const float x = xs[k * ld + c];
          t[0] = fmaf(g.x, x, t[0]); t[1] = fmaf(g.y, x, t[1]); t[2] = fmaf(g.z, x, t[2]); t[3] = fmaf(g.w, x, t[3]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += t[r];
      }
    },
    [&](int u, const float (&v)[4]) {
      const int j = u / d, c = u - j * d;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (j * 4 + r < V) store_as(a.gw, (int64_t)(j * 4 + r) * d + c, v[r], a.dtype);
    });
}

}  // namespace psb

using namespace psb;

namespace {

constexpr int kMaxBlocks = 148 * 8;           // of the pass that finds the largest magnitudes, for either operand

// where things lie in the workspace; everything is 256-byte aligned
struct LossPlan {
  int planes, pack_x, pack_w, parts, per_tile, keep, piece, together;
  int tiny, tiny_ld, tiny_ldg, tiny_smem;     // CTAs of k_loss_tiny, 0: the general way
  Tiling score, gx, gw;                       // gx, gw: of the kept classes, or of a piece
  int64_t dp, ldg, x_plane, w_plane, g_plane;
  int64_t scales, maxima, lse, target, x, w, part, g, gx_acc, gw_acc, total;
};

// what a plan depends on: sizes, types and alignment
struct LossKey {
  int n, V, d, dtype, want_grad, want_gx, keep_mb, pack_x, pack_w;
  bool operator==(const LossKey& o) const {
    return n == o.n && V == o.V && d == o.d && dtype == o.dtype && want_grad == o.want_grad && want_gx == o.want_gx && keep_mb == o.keep_mb &&
           pack_x == o.pack_x && pack_w == o.pack_w;
  }
};
LossKey loss_key(const LossArgs& a) {
  auto direct = [&](const void* t, int64_t ld) {
    return a.dtype != kF32 && (ld & 7) == 0 && (reinterpret_cast<uintptr_t>(t) & 15) == 0 && ld >= a.d;
  };
  return LossKey{a.n, a.V, a.d, a.dtype, a.want_grad, a.gx != nullptr, a.keep_mb, !direct(a.x, a.ldx), !direct(a.w, a.ldw)};
}

// One launch where rows, classes and scores fit into shared memory and the multiplications do not take the CUDA cores longer than
// the general way takes for its launches.
bool tiny_plan(LossPlan& p, const LossKey& a) {
  const int64_t work = (int64_t)a.n * a.V * (a.d < kTinyWork ? a.d : kTinyWork);
  if (a.n > kTinyRows || a.V > kTinyRows || work > kTinyWork) return false;
  const int64_t ld = ((int64_t)a.d + 3) / 4 | 1, n4 = ((int64_t)a.n + 3) / 4, v4 = ((int64_t)a.V + 3) / 4;       // in fours
  const int64_t bytes = ((n4 + v4) * 4 * ld + n4 * 4 * v4) * 16;
  if (bytes > kTinySmem) return false;
  p.tiny = work <= kTinyAlone ? 1 : kTinyCtas;
  p.tiny_ld = (int)ld * 4; p.tiny_ldg = (int)v4 * 4; p.tiny_smem = (int)bytes;
  return true;
}

LossPlan make_loss_plan(const LossKey& a) {
  LossPlan p = {};
  if (tiny_plan(p, a)) return p;
  p.planes = a.dtype == kF32 ? 2 : 1;
  p.dp = ((int64_t)a.d + 7) / 8 * 8;
  p.pack_x = a.pack_x;
  p.pack_w = a.pack_w;
  p.score = choose_tiling(1, a.n, a.V, a.d, p.planes, false, 1);
  const int cols = tiling_cols(p.score.kind);
  p.per_tile = tiling_parts(p.score.kind);
  p.parts = p.per_tile * ((a.V + cols - 1) / cols);
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  p.scales = take(sizeof(Scales));
  p.maxima = take(2 * kMaxBlocks * 4);
  p.lse = take((int64_t)a.n * 4);
  p.target = take((int64_t)a.n * 4);
  p.x_plane = (int64_t)a.n * p.dp;
  if (p.pack_x || a.want_grad) p.x = take(p.x_plane * 2 * p.planes);
  p.w_plane = (int64_t)a.V * p.dp;
  if (p.pack_w) p.w = take(p.w_plane * 2 * p.planes);
  p.part = take((int64_t)p.parts * a.n * 8);
  if (a.want_grad) {
    int64_t len = ((int64_t)a.keep_mb << 20) / ((int64_t)a.n * 2 * p.planes) / 256 * 256;
    if (len < 256) len = 256;
    p.keep = p.piece = (int)(len < a.V ? len : a.V);
    p.ldg = ((int64_t)p.piece + 7) / 8 * 8;
    p.g_plane = (int64_t)a.n * p.ldg;
    p.g = take(p.g_plane * 2 * p.planes);
    const bool pieces = p.piece < a.V;
    p.gw = choose_tiling(1, p.piece, a.d, a.n, p.planes, false, pieces ? 1 : 16);
    p.gx = choose_tiling(1, a.n, a.d, p.piece, p.planes, false, pieces ? 1 : 64);
    // both in one launch where their tiles, of one kind, are one round: a launch less, and a third of the SMs does not wait
    if (a.want_gx && !pieces && (p.gw.kind == kOne128 || p.gw.kind == kOne64)) {
      const Tiling t = choose_tiling(1, a.n, a.d, p.piece, p.planes, false, 64, 1, p.gw.kind);
      auto tiles = [&](const Tiling& u, int64_t M) { return (M + 127) / 128 * ((a.d + tiling_cols(u.kind) - 1) / tiling_cols(u.kind)) * u.splits; };
      if (tiles(p.gw, a.V) + tiles(t, a.n) <= 148) {
        p.together = 1;
        p.gx = t;
      }
    }
    if (a.want_gx && (p.gx.splits > 1 || pieces)) p.gx_acc = take((int64_t)p.gx.splits * a.n * a.d * 4);
    if (p.gw.splits > 1) p.gw_acc = take((int64_t)p.gw.splits * a.V * a.d * 4);
  }
  p.total = at;
  return p;
}

// The search for tiles takes microseconds, twice a call: a thread keeps the plans of the sizes that it met last.
LossPlan loss_plan(const LossArgs& a) {
  struct Entry { LossKey key; LossPlan plan; bool used; };
  static thread_local Entry kept[16] = {};
  const LossKey k = loss_key(a);
  Entry& e = kept[((unsigned)k.n * 31u + (unsigned)k.V * 7u + (unsigned)k.d * 13u + (unsigned)k.want_grad) % 16u];
  if (!e.used || !(e.key == k)) e = Entry{k, make_loss_plan(k), true};
  return e.plan;
}

unsigned blocks_for(int64_t threads, int64_t most) {
  const int64_t b = (threads + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > most ? most : b);
}

bool loss_args_ok(const LossArgs& a) {
  return a.n > 0 && a.V > 0 && a.d > 0 && a.dtype >= kF32 && a.dtype <= kF16 && a.V <= (1 << 30) && a.n <= (1 << 30) && a.d <= (1 << 30) &&
         a.keep_mb >= 0;
}

template <typename T>
int tiny_launch(cudaStream_t stream, const LossPlan& p, const TinyArgs& q) {
  int dev = 0;
  if (sm_count(&dev) <= 0) return (int)cudaErrorInvalidDevice;
  static bool attr[kMaxDevices] = {};
  if (!attr[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k_loss_tiny<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTinySmem);
    if (e != cudaSuccess) return (int)e;
    attr[dev] = true;
  }
  Chain chain{stream};
  return chain.launch(k_loss_tiny<T>, dim3((unsigned)p.tiny), kTinyThreads, (size_t)p.tiny_smem, p.tiny, q);
}

// A gradient [M, N], contiguous, from a product, whole or split.
struct Gradient {
  Gemm16Args g;
  Operand16 a, b;
  EpiGrad::Params e;
};
int prepare(Gradient& q, const Tiling& t) {
  q.g.splits = t.splits;
  q.g.kb_split = t.splits > 1 ? t.kb_split : (q.g.K + kG16K - 1) / kG16K;
  q.e.M = q.g.M; q.e.N = q.g.N;
  if (t.splits > 1) { q.e.slot = (int64_t)q.g.M * q.g.N; q.e.write = 1; q.e.read = 0; }
  q.e.by_map = !q.e.write && !q.e.read && q.e.dtype != kF32 && (q.g.N & 7) == 0 && (reinterpret_cast<uintptr_t>(q.e.out) & 15) == 0;
  return q.e.by_map ? make_out_map(&q.e.map, Operand16{q.e.out, q.g.M, q.g.N, q.g.N, 0, 1}, q.e.dtype == kBF16) : 0;
}
int add_splits(Chain& chain, const Gradient& q) {
  if (q.g.splits == 1) return 0;
  const EpiGrad::Params& e = q.e;
  return chain.launch(k_loss_sum, dim3(blocks_for(e.slot, 148 * 8)), 256, 0, 1, e.acc, q.g.splits, e.slot, e.slot, e.out, e.dtype);
}
// One gradient, or two in one launch
int gradient(Chain& chain, int planes, int kind, const Gradient& q) {
  const int r = product16<EpiGrad>(chain, planes, kind, q.g, q.a, q.b, q.e);
  return r ? r : add_splits(chain, q);
}
int gradients(Chain& chain, int planes, int kind, const Gradient (&q)[2]) {
  Launch16<EpiGrad, 2> l = {{q[0].g, q[1].g}, {q[0].e, q[1].e}};
  const Operand16 a[2] = {q[0].a, q[1].a}, b[2] = {q[0].b, q[1].b};
  int r = products16<EpiGrad>(chain, planes, kind, l, a, b);
  if (r == 0) r = add_splits(chain, q[0]);
  return r ? r : add_splits(chain, q[1]);
}

}  // namespace

extern "C" {

// bytes of workspace that the call with these arguments needs (-1: arguments out of range)
int64_t psb_softmax_loss_workspace(const LossArgs* a) { return loss_args_ok(*a) ? loss_plan(*a).total : -1; }

// Returns 0, a CUDA error, or -1 without the driver's entry point for tensor maps.
int psb_softmax_loss(const LossArgs* ap, cudaStream_t s) {
  const LossArgs& a = *ap;
  if (!loss_args_ok(a)) return (int)cudaErrorInvalidValue;
  const LossPlan p = loss_plan(a);
  if (p.tiny) {
    const TinyArgs q{a, p.tiny_ld, p.tiny_ldg, p.tiny};
    return a.dtype == kF32 ? tiny_launch<float>(s, p, q) : a.dtype == kBF16 ? tiny_launch<__nv_bfloat16>(s, p, q) : tiny_launch<__half>(s, p, q);
  }
  if (p.total > a.ws_bytes || (reinterpret_cast<uintptr_t>(a.ws) & 255)) return (int)cudaErrorInvalidValue;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.ws);
  Scales* found = reinterpret_cast<Scales*>(ws + p.scales);
  uint32_t* maxima = reinterpret_cast<uint32_t*>(ws + p.maxima);
  float *lse = reinterpret_cast<float*>(ws + p.lse), *target = reinterpret_cast<float*>(ws + p.target);
  uint16_t *xb = reinterpret_cast<uint16_t*>(ws + p.x), *wb = reinterpret_cast<uint16_t*>(ws + p.w), *gb = reinterpret_cast<uint16_t*>(ws + p.g);
  float2* part = reinterpret_cast<float2*>(ws + p.part);
  Chain chain{s};
  int r = 0;

  ScaleRef scale{{0, 0, a.dtype == kBF16 ? 0 : 13}, nullptr};       // without coefficients the largest is 1
  if (a.dtype == kF32 || (a.dtype == kF16 && a.coef != nullptr && a.want_grad)) scale.found = found;
  if (scale.found != nullptr && a.dtype == kF16) r = chain.launch(k_loss_coef, dim3(1), 256, 0, 1, a.coef, a.y, a.n, a.V, found);
  unsigned mx = 0, mw = 0;
  const bool small = ((int64_t)a.n + a.V) * a.d <= 32768;      // 128 KB: 32 values a thread, less than a launch
  if (a.dtype == kF32 && !small) {
    mx = blocks_for((int64_t)a.n * ((a.d + 3) / 4), kMaxBlocks);
    mw = blocks_for((int64_t)a.V * ((a.d + 3) / 4), kMaxBlocks);
    r = chain.launch(k_loss_absmax, dim3(mx + mw), 256, 0, 1, (const float*)a.x, a.ldx, (const float*)a.w, a.ldw, a.n, a.V, a.d, a.y, (int)mx, maxima);
  }
  if (r) return r;
  if (p.pack_x || p.pack_w) {
    const PackArgs px{a.x, a.n, a.ldx, xb, p.dp, p.x_plane}, pw{a.w, a.V, a.ldw, wb, p.dp, p.w_plane};
    const unsigned bx = p.pack_x ? blocks_for((int64_t)a.n * (p.dp / 8), 148 * 8) : 0, bw = p.pack_w ? blocks_for((int64_t)a.V * (p.dp / 8), 148 * 8) : 0;
    auto pack = [&](auto kernel) {
      return chain.launch(kernel, dim3(bx + bw), 256, 0, 1, px, pw, a.d, a.y, a.n, a.V, a.coef, (int)bx, small ? nullptr : maxima, (int)mx, (int)mw, found);
    };
    r = a.dtype == kF32 ? pack(k_loss_pack<float>) : a.dtype == kBF16 ? pack(k_loss_pack<__nv_bfloat16>) : pack(k_loss_pack<__half>);
    if (r) return r;
  }

  // scores
  const Operand16 x = p.pack_x ? Operand16{xb, a.n, a.d, p.dp, p.x_plane, p.planes} : Operand16{a.x, a.n, a.d, a.ldx, 0, 1};
  const Operand16 w = p.pack_w ? Operand16{wb, a.V, a.d, p.dp, p.w_plane, p.planes} : Operand16{a.w, a.V, a.d, a.ldw, 0, 1};
  Gemm16Args g = {};
  g.batch = 1; g.splits = 1; g.bf16 = a.dtype == kBF16; g.status = a.status;
  g.M = a.n; g.N = a.V; g.K = a.d;
  g.kb_split = (a.d + kG16K - 1) / kG16K;
  EpiScore::Params es = {};
  es.part = part; es.target = target; es.y = a.y; es.scale = scale; es.n = a.n; es.V = a.V; es.parts = p.parts; es.per_tile = p.per_tile; es.keep = p.keep;
  if (a.want_grad && (r = make_out_map(&es.e, Operand16{gb, a.n, p.keep, p.ldg, p.g_plane, p.planes}, 0)) != 0) return r;
  if ((r = product16<EpiScore>(chain, p.planes, p.score.kind, g, x, w, es)) != 0) return r;

  // losses, and G of the kept classes
  JoinArgs j = {};
  j.part = part; j.target = target; j.y = a.y; j.coef = a.coef; j.lse = lse; j.loss = a.loss; j.scale = scale;
  j.n = a.n; j.V = a.V; j.d = a.d; j.parts = p.parts; for (j.shift = 5; tiling_cols(p.score.kind) / p.per_tile > 1 << j.shift; ++j.shift) {} j.keep = p.keep; j.dtype = a.dtype; j.status = a.status;
  if (a.want_grad) {
    j.g = gb; j.ldg = p.ldg; j.plane = p.g_plane;
    if (!p.pack_x) { j.x = reinterpret_cast<const uint16_t*>(a.x); j.x_out = xb; j.ldx = a.ldx; j.ldxo = p.dp; }
  }
  if (p.parts <= 64 && a.V <= 2048) {           // a warp a row; with and without gradients alike, so that losses are the same
    r = chain.launch(k_loss_rows<32>, dim3((unsigned)(a.n + 7) / 8, 1), 256, 0, 1, j);
  } else {
    int64_t share = a.want_grad ? (148 * 6 + a.n - 1) / a.n : 1, most = ((int64_t)p.keep + 8191) / 8192;
    if (share > most) share = most < 1 ? 1 : most;
    r = chain.launch(k_loss_rows<256>, dim3((unsigned)a.n, (unsigned)share), 256, 0, 1, j);
  }
  if (r || !a.want_grad) return r;

  const Operand16 xz{xb, a.n, a.d, p.dp, p.x_plane, p.planes};      // rows without a class are zeros
  const int64_t es_out = a.dtype == kF32 ? 4 : 2;
  for (int v0 = 0; v0 < a.V; v0 += p.piece) {
    const int len = a.V - v0 < p.piece ? a.V - v0 : p.piece;
    const Operand16 gop{gb, a.n, len, p.ldg, p.g_plane, p.planes};
    if (v0 > 0) {                              // beyond the kept classes: scores once more
      Gemm16Args gs = g;
      gs.N = len; gs.b_n0 = v0;
      EpiG::Params eg = {};
      if ((r = make_out_map(&eg.g, gop, a.dtype == kBF16)) != 0) return r;
      eg.lse = lse; eg.coef = a.coef; eg.y = a.y; eg.scale = scale; eg.n = a.n; eg.V = a.V; eg.len = len; eg.v0 = v0; eg.dtype = a.dtype;
      if ((r = product16<EpiG>(chain, p.planes, choose_tiling(1, a.n, len, a.d, p.planes, false, 1).kind, gs, x, w, eg)) != 0) return r;
    }
    EpiGrad::Params e = {};
    e.scale = scale; e.dtype = a.dtype;
    Gradient q[2];
    // gw[v0.., :] = Gᵀ x
    q[0] = Gradient{g, gop, xz, e};
    q[0].g.M = len; q[0].g.N = a.d; q[0].g.K = a.n; q[0].g.a_mn = q[0].g.b_mn = 1;
    q[0].e.out = reinterpret_cast<uint8_t*>(a.gw) + (int64_t)v0 * a.d * es_out;
    if (p.gw.splits > 1) q[0].e.acc = reinterpret_cast<float*>(ws + p.gw_acc);
    if ((r = prepare(q[0], p.gw)) != 0) return r;
    if (!p.together && (r = gradient(chain, p.planes, p.gw.kind, q[0])) != 0) return r;
    if (a.gx == nullptr) continue;
    // gx += G w[v0.., :]
    q[1] = Gradient{g, gop, w, e};
    q[1].g.M = a.n; q[1].g.N = a.d; q[1].g.K = len; q[1].g.b_k0 = v0; q[1].g.b_mn = 1;
    q[1].e.out = a.gx; q[1].e.with_w = 1;
    if (p.gx.splits > 1 || p.piece < a.V) q[1].e.acc = reinterpret_cast<float*>(ws + p.gx_acc);
    if (p.piece < a.V) { q[1].e.read = v0 > 0; q[1].e.write = v0 + len < a.V; }
    if ((r = prepare(q[1], p.gx)) != 0) return r;
    r = p.together ? gradients(chain, p.planes, p.gx.kind, q) : gradient(chain, p.planes, p.gx.kind, q[1]);
    if (r) return r;
  }
  return 0;
}

}  // extern "C"
