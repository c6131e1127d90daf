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
// is known then), for as many classes as the workspace holds; the second kernel (a third for fp32) turns it into G in place, with
// one factor a part.  Making the scores once costs 6nVd operations instead of 8nVd, for a pass over 2 bytes an element
// (8192 rows, 131,072 classes, 2048 wide: 3.2 ms less for 0.85).  Classes beyond the workspace come in pieces, whose scores
// are made again.  gw of a piece is complete, gx is summed over the pieces in fp32.  Sums have a fixed order: results do not
// vary from run to run.
//
// Bound by the tensor cores: bf16 scores of 4096 rows against 131,072 classes, 1024 wide, take 785 to 810 us, 0.8 of the rate of a
// plain cuBLAS product; 8192 x 131,072 x 2048 with gradients takes 10.4 to 10.9 ms where the products alone, at its sustained rate, take 9.5.
//
// Scores, maxima, sums and losses are fp32 (in units of log2 e: 2^x is the hardware's exponential).  The exponentials keep 11
// bits (two planes for fp32: 22); the label's entry of G, where they would cancel, is made from the label's score in fp32.
// G is rounded to the operands' type: bf16 for bf16; fp16 for fp16, scaled by a power of two so that the largest
// coefficient is near 2^13; two planes of fp16 for fp32, where x and w are such planes too.
//
// Scales of fp32 operands.  Every row of x and every class of w has a power of two of its own, 2^kx_i and 2^kw_j, that brings its
// largest element to [2^14, 2^15); the epilogues of the scores undo both.  (One power for all of x lets one large row take the bits
// of all the others: 64 rows, one times 10^10, and the others' losses are 0.1 off.)  The two gradient products sum over different
// indices and take G scaled differently:
//   gx_i = 2^{a_i} Σ_j (G_ij 2^{-kw_j} 2^{-a_i}) (2^{kw_j} w_j)      a_i of a row, from the row's largest G_ij 2^{-kw_j}
//   gw_j = 2^{b_t} Σ_i (G_ij 2^{-kx_i} 2^{-b_t}) (2^{kx_i} x_i)      b_t of a part of a tile's classes, from the largest G_ij 2^{-kx_i} there
// so that either sum keeps 22 bits of terms down to 2^-17 of its largest, and a unit of 2^-38 of that below.  The maxima follow
// from the parts' maxima once a row's log-sum-exp is known.
#include "gemm16.cuh"

namespace psb {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kExpScale = 15;                 // exponentials relative to their maximum are kept times 2^15

enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// Exponent of the scale of G with 16-bit operands: 0 for bf16; for fp16 it is known where there are no coefficients, else the
// device finds it.
struct ScaleRef {
  int fixed;
  const int* found;            // null: as fixed
  __device__ __forceinline__ int get() const { return found != nullptr ? *found : fixed; }
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
// 2^e in two factors of the same direction: the power may lie outside fp32 where what it scales does not leave it
struct Pow2 {
  float a, b;
  __device__ __forceinline__ explicit Pow2(int e) : a(pow2i(e / 2)), b(pow2i(e - e / 2)) {}
  __device__ __forceinline__ float operator*(float v) const { return v * a * b; }
};
__device__ __forceinline__ int exponent(float v) { return (int)(__float_as_uint(v) >> 23 & 255u) - 127; }       // of a normal number
// The exponent of a part's scale from that of its largest G_ij 2^{-kx_i}; no row has any: 0
constexpr int kScaleTop = 14, kNoRow = -(1 << 30);
__device__ __forceinline__ int part_scale(int largest) { return largest == kNoRow ? 0 : largest - kScaleTop; }
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
k_loss_coef(const float* __restrict__ coef, const int64_t* __restrict__ y, int n, int V, int* out) {
  pdl_wait();
  const uint32_t top = coef_max(coef, y, n, V);
  if (threadIdx.x == 0) *out = scale_exp(top, 13);
}

struct PackArgs {
  const void* a;               // rows of `cols` elements, any stride and alignment
  int64_t rows, ld;
  uint16_t* out;               // operand planes [plane][row][ldo]
  int64_t ldo, plane;
};
// 16-bit operands into rows of their own: blocks 0..bx-1 copy x, the others w (either may have no blocks).  Rows of x without a
// class become zeros, whatever they held.
template <typename T>
__global__ void __launch_bounds__(256)
k_loss_pack(PackArgs px, PackArgs pw, int cols, const int64_t* __restrict__ y, int V, int bx) {
  pdl_wait();
  const bool is_x = (int)blockIdx.x < bx;
  const PackArgs& p = is_x ? px : pw;
  const int64_t nb = is_x ? bx : gridDim.x - bx, b = is_x ? blockIdx.x : blockIdx.x - bx;
  const T* a = reinterpret_cast<const T*>(p.a);
  if (((reinterpret_cast<uintptr_t>(a) & 15) | (p.ld & 7)) != 0) {
    // rows of any alignment: a warp a row, two columns a thread, so that loads and stores are pieces of one row
    const int64_t warps = nb * 8;
    for (int64_t r = b * 8 + (threadIdx.x >> 5); r < p.rows; r += warps) {
      const T* src = a + r * p.ld;
      uint16_t* dst = p.out + r * p.ldo;
      const bool none = is_x && !has_class(y[r], V);
#pragma unroll 4
      for (int c = (threadIdx.x & 31) * 2; c < (int)p.ldo; c += 64) {
        const T u = !none && c < cols ? src[c] : T(0), v = !none && c + 1 < cols ? src[c + 1] : T(0);
        *reinterpret_cast<uint32_t*>(dst + c) = (uint32_t)*reinterpret_cast<const uint16_t*>(&u) | (uint32_t)*reinterpret_cast<const uint16_t*>(&v) << 16;
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
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? src[j] : T(0);
    }
    *reinterpret_cast<uint4*>(p.out + r * p.ldo + c) = *reinterpret_cast<uint4*>(v);
  }
}

// fp32 operands into planes, the rows of x and then those of w: kLanes threads (a warp, or the block of 256) find a row's largest
// finite magnitude, write the power of two that undoes its scale, and split the row.  Rows of x without a class become
// zeros.  A row of zeros has the largest scale, so that it has no part in maxima over rows.
template <int kLanes>
__global__ void __launch_bounds__(256)
k_loss_planes(PackArgs px, PackArgs pw, int cols, const int64_t* __restrict__ y, int n, int V, float* __restrict__ fx, float* __restrict__ fw,
              int* __restrict__ largest, int parts) {
  pdl_wait();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < parts; i += gridDim.x * 256) largest[i] = kNoRow;
  const int ln = threadIdx.x % kLanes;
  const int64_t rows = (int64_t)n + V;
  for (int64_t r = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; r < rows; r += (int64_t)gridDim.x * (256 / kLanes)) {
    const bool is_x = r < n;
    const PackArgs& p = is_x ? px : pw;
    const int64_t row = is_x ? r : r - n;
    const float* src = reinterpret_cast<const float*>(p.a) + row * p.ld;
    uint16_t* dst = p.out + row * p.ldo;
    const int d = is_x && !has_class(y[row], V) ? 0 : cols;
    const bool vec = ((reinterpret_cast<uintptr_t>(p.a) & 15) | (p.ld & 3)) == 0;
    uint32_t top = 0;
    if (vec) {
#pragma unroll 4
      for (int c = ln * 4; c < d; c += kLanes * 4) {
        if (c + 4 <= d) {
          const float4 v = *reinterpret_cast<const float4*>(src + c);
          top = max(max(top, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
        } else {
          for (int j = c; j < d; ++j) top = max(top, finite_bits(src[j]));
        }
      }
    } else {
#pragma unroll 4
      for (int c = ln; c < d; c += kLanes) top = max(top, finite_bits(src[c]));
    }
    top = kLanes == 32 ? __reduce_max_sync(0xffffffffu, top) : block_max_u32(top);
    const int k = top == 0 ? 126 : scale_exp(top, kScaleTop);
    const float s = pow2i(k);
    if (ln == 0) (is_x ? fx : fw)[row] = pow2i(-k);
    if (vec) {
#pragma unroll 4
      for (int c = ln * 4; c < (int)p.ldo; c += kLanes * 4) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c + 4 <= d) v = *reinterpret_cast<const float4*>(src + c);
        else {
          if (c < d) v.x = src[c];
          if (c + 1 < d) v.y = src[c + 1];
          if (c + 2 < d) v.z = src[c + 2];
        }
        *reinterpret_cast<uint2*>(dst + c) = make_uint2(pair16<kFmtPlanes>(v.x * s, v.y * s, false), pair16<kFmtPlanes>(v.z * s, v.w * s, false));
        *reinterpret_cast<uint2*>(dst + p.plane + c) = make_uint2(pair16<kFmtPlanes>(v.x * s, v.y * s, true), pair16<kFmtPlanes>(v.z * s, v.w * s, true));
      }
    } else {                                  // two columns a thread, so that loads and stores are pieces of one row
#pragma unroll 4
      for (int c = ln * 2; c < (int)p.ldo; c += kLanes * 2) {
        const float u = c < d ? src[c] * s : 0.f, v = c + 1 < d ? src[c + 1] * s : 0.f;
        *reinterpret_cast<uint32_t*>(dst + c) = pair16<kFmtPlanes>(u, v, false);
        *reinterpret_cast<uint32_t*>(dst + p.plane + c) = pair16<kFmtPlanes>(u, v, true);
      }
    }
  }
}

// ------------------------------------------------------------------ epilogues
// Each row's maximum and Σ 2^(s−m) over a part of a tile's classes, the score of its label, in units of log2 e, and the
// exponentials that are kept.  With planes, the largest 2^(s−m) 2^{-kw} and the largest 2^(s−m) of the part as well, both without
// the label's class: where its softmax is near 1, its G is near 0.
struct EpiScore {
  static constexpr int kLongK = 4096;
  struct Params {
    CUtensorMap e;             // exponentials [plane][n][keep]
    float2* part;              // [n][per_tile · class tiles]; null: the exponentials alone, of classes from v0 on
    float2* widest;            // [n][the same]
    float* target;             // [n]
    const int64_t* y;
    const float *fx, *fw;      // powers of two that undo the scales of rows and classes
    int n, V, parts, per_tile, keep, v0;
  };
  template <int kPart>
  static __device__ __forceinline__ void ahead(const Params&, const Tile16&, int, int, int) {}
  template <int kPlanes, int kPart, class Stage, class Sums, class Done>
  static __device__ __forceinline__ void run(const Params& p, const Gemm16Args&, const Tile16& w, int row0, int col0, int part, Stage& st,
                                             const Sums& sums, Done done) {
    constexpr bool kScaled = kPlanes == 2;
    const int row = row0 + st.lane;
    int64_t lab = -1;
    if (row < p.n) lab = p.y[row] < p.V ? p.y[row] - p.v0 : -1;
    // A row's factor comes before the class's where it is below 1 and after it elsewhere: no product leaves fp32 on the way to a score
    // that does not.
    float before = kLog2e, after = 1.f;
    if (kScaled && row < p.n) {
      const float f = p.fx[row];
      before = kLog2e * fminf(f, 1.f);
      after = fmaxf(f, 1.f);
    }
    // 32 scores; without planes they are not in units of log2 e yet
    auto scores = [&](int c, float (&v)[32], float (&f)[32]) {
      sums.load(c, v);
      if constexpr (kScaled) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 t = *reinterpret_cast<const float4*>(p.fw + p.v0 + col0 + c + j);       // behind the last class lies padding
          f[j] = t.x; f[j + 1] = t.y; f[j + 2] = t.z; f[j + 3] = t.w;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __fmul_rn(v[j], before) * f[j] * after;
      }
    };
    auto scaled = [](float v) { return kScaled ? v : __fmul_rn(v, kLog2e); };
    const int classes = p.V - p.v0;
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kPart; c += 32) {
      float v[32], f[32];
      scores(c, v, f);
      const int left = classes - (col0 + c);
      if (left >= 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = j < left ? fmaxf(top, v[j]) : top;
      }
    }
    // without a finite score the reference is 0: 2^(-inf) is 0 and nothing is subtracted from an infinity
    const float m = scaled(top), ref = top == -INFINITY ? 0.f : m;
    float s = 0.f;
    float2 widest = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int c = 0; c < kPart; c += 32) {
      float v[32], f[32];
      scores(c, v, f);
      if (c + 32 >= kPart) done();
      const int col = col0 + c, left = classes - col;
      if (left <= 0) continue;
      const int at = lab >= col && lab < col + 32 ? (int)(lab - col) : -1;
      if (p.part != nullptr && at >= 0) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) t = j == at ? v[j] : t;
        p.target[row] = scaled(t);
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        // product and difference rounded apart, as those of the maximum and of the label are: a row whose class is certain has
        // a loss of 0, not of a rounding
        v[j] = ex2(__fsub_rn(scaled(v[j]), ref));
        if (left < 32) v[j] = j < left ? v[j] : 0.f;
        s += v[j];
      }
      if constexpr (kScaled) {
        if (p.widest != nullptr) {
          if (__any_sync(0xffffffffu, at >= 0)) {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = j == at ? 0.f : f[j];
#pragma unroll
            for (int j = 0; j < 32; ++j) widest.y = j == at ? widest.y : fmaxf(widest.y, v[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) widest.y = fmaxf(widest.y, v[j]);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) widest.x = fmaxf(widest.x, v[j] * f[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= (float)(1 << kExpScale);
      if (col < p.keep) st.template store<kPlanes == 2 ? kFmtPlanes : kFmtF16>(&p.e, v, row0, col, 0, false);
    }
    if (row < p.n && p.part != nullptr) {
      const int64_t at = (int64_t)row * p.parts + w.tn * p.per_tile + part;
      p.part[at] = make_float2(top == -INFINITY ? top : m, s);
      if (kScaled && p.widest != nullptr) p.widest[at] = widest;
    }
  }
};

// G of a piece of the classes, in the operands' 16-bit type, from scores made again
struct EpiG {
  static constexpr int kLongK = EpiScore::kLongK;
  struct Params {
    CUtensorMap g;             // [n][len]
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
    const int row = row0 + st.lane;
    float c = 0.f, lse = 0.f;
    int64_t lab = -1;
    if (row < p.n && has_class(p.y[row], p.V)) {
      lab = p.y[row] - p.v0;
      c = (p.coef != nullptr ? p.coef[row] : 1.f) * pow2i(p.scale.get());
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
      for (int j = 0; j < 32; ++j) v[j] = none ? 0.f : c * (ex2(fmaf(v[j], kLog2e, -lse)) - (at == j ? 1.f : 0.f));
      if (p.dtype == kBF16) st.template store<kFmtBF16>(&p.g, v, row0, col, 0, false);
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
  static constexpr int kLongK = 32768;
  struct Params {
    CUtensorMap map;           // of the result, where it is 16-bit and aligned
    void* out;
    float* acc;
    int64_t slot;
    ScaleRef scale;            // without planes: of G
    const int* exps;           // with planes: a power of two of the product's rows, of 2^exp_shift of them from row exp_first on
    int exp_first, exp_shift, exp_parts;       // exp_parts: exps are the parts' largest
    int M, N, dtype, by_map;
    int read, write;           // acc is added to the product; the sum goes to acc instead of the result
  };
  template <int kPart>
  static __device__ __forceinline__ void ahead(const Params& p, const Tile16& w, int row, int col, int lane) {
    if (p.read && row + lane < p.M) prefetch_l2<kPart>(p.acc + w.split * p.slot + (int64_t)(row + lane) * p.N, col, p.N);
  }
  template <int kPlanes, int kPart, class Stage, class Sums, class Done>
  static __device__ __forceinline__ void run(const Params& p, const Gemm16Args&, const Tile16& w, int row0, int col0, int, Stage& st,
                                             const Sums& sums, Done done) {
    int e = 0;
    if constexpr (kPlanes == 1) {
      e = -p.scale.get();
    } else if (row0 + st.lane < p.M) {
      e = p.exps[(p.exp_first + row0 + st.lane) >> p.exp_shift];
      if (p.exp_parts) e = part_scale(e);
    }
    const Pow2 scale(e);
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
    __syncthreads();                          // of the row before
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
    __syncthreads();
    a = sh[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) a = join(a, sh[i]);
  }
  return a;
}

// What the gradients of fp32 operands need of a row: the maximum and the rest of its log-sum-exp (log2), p − 1 of its label's
// softmax p, and its coefficient c = mant · 2^e with the scales that G takes:  c 2^{-a_i} = to_x,  c 2^{-kx_i} = mant · 2^to_w.
struct RowStat {
  float top, rest, at_label, mant, to_x;
  int to_w, pad[2];
};

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
  // fp32
  const float2* widest;
  const float *fx, *fw;
  RowStat* stat;               // null: the losses alone
  int *row_exp, *largest;      // a_i; of a part's scale
  uint16_t* g2;                // g becomes G for gx, this is G for gw
  int v0, len;                 // the classes that g holds
};
// 16-bit operands: a row's log-sum-exp (log2) and loss and, in place, its kept exponentials to G.  kLanes threads a row; blockIdx.y shares
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
  const int kg = p.scale.get();
  const float cg = c * pow2i(kg), at_label = cg * (ex2((target - a.x) - l2) - 1.f);
  const float shift = (float)kExpScale + l2;
  uint16_t* g = p.g + (int64_t)row * p.ldg;
  // four eights a thread at a time: their loads do not wait for one another
  const int step = gridDim.y * kLanes * 8;
  for (int first = (blockIdx.y * kLanes + ln) * 8; first < p.keep; first += 4 * step) {
    uint4 h[4];
    float f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int col = first + k * step;
      if (col >= p.keep) break;
      h[k] = *reinterpret_cast<const uint4*>(g + col);
      f[k] = part[col >> p.shift].x;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int col = first + k * step;
      if (col >= p.keep) break;
      const float scale = cg * ex2((f[k] - a.x) - shift);
      const int at = lab >= col && lab < col + 8 ? (int)(lab - col) : -1;
      uint32_t hs[4] = {h[k].x, h[k].y, h[k].z, h[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hs[i]));
        v.x = ok ? (at == 2 * i ? at_label : v.x * scale) : 0.f;
        v.y = ok ? (at == 2 * i + 1 ? at_label : v.y * scale) : 0.f;
        hs[i] = p.dtype == kBF16 ? pair16<kFmtBF16>(v.x, v.y, false) : pair16<kFmtF16>(v.x, v.y, false);
      }
      *reinterpret_cast<uint4*>(g + col) = make_uint4(hs[0], hs[1], hs[2], hs[3]);
    }
  }
}

// fp32 operands: rows' log-sum-exp and loss, the scale of their G for gx, and the scales of G for gw.  kLanes threads a row, row
// after row, so that a block offers its largest of a part once (34 parts of 8162 rows: 47 us with an atomic for every row).
constexpr int kJoinParts = 4096;              // whose largest a block keeps; beyond them rows are few
template <int kLanes>
__global__ void __launch_bounds__(256)
k_loss_join(const __grid_constant__ JoinArgs p) {
  __shared__ int mine[kJoinParts];
  __shared__ float sh[8];
  const int ln = threadIdx.x % kLanes, kept = p.stat == nullptr ? 0 : p.parts < kJoinParts ? p.parts : kJoinParts;
  for (int t = threadIdx.x; t < kept; t += 256) mine[t] = kNoRow;
  pdl_wait();
  __syncthreads();
  for (int row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; row < p.n; row += gridDim.x * (256 / kLanes)) {
    const float2* part = p.part + (int64_t)row * p.parts;
    const float2 a = join_row<kLanes>(part, p.parts, ln);
    const float rest = log2f(a.y);
    const int64_t lab = p.y[row];
    const bool ok = has_class(lab, p.V);
    const float c = ok ? (p.coef != nullptr ? p.coef[row] : 1.f) : 0.f;
    const float target = ok ? p.target[row] : 0.f;
    if (ln == 0) {
      if (lab != -1 && !ok) set_status(p.status, kBadIndex, (uint32_t)row, (uint32_t)lab);
      p.loss[row] = ok ? c * (kLn2 * ((a.x - target) + rest)) : 0.f;
    }
    if (p.stat == nullptr) continue;
    // NaN compares as false and is left out of the maxima
    const float at_label = ok ? ex2((target - a.x) - rest) - 1.f : 0.f, at_log = log2f(fabsf(at_label)), c_log = log2f(fabsf(c));
    const int fx = exponent(p.fx[row]);
    auto offer = [&](int t, float v) {
      v += c_log + (float)fx;
      if (!(v > -1000.f)) return;
      const int e = (int)floorf(v < 1000.f ? v : 1000.f);
      int* to = t < kJoinParts ? mine + t : p.largest + t;
      if (e > *reinterpret_cast<volatile int*>(to)) atomicMax(to, e);
    };
    float top = -INFINITY;
    const float2* widest = p.widest + (int64_t)row * p.parts;
    if (ok)
      for (int t = ln; t < p.parts; t += kLanes) {
        const float v = (part[t].x - a.x) - rest;
        const float2 u = widest[t];
        top = fmaxf(top, v + log2f(u.x));
        offer(t, v + log2f(u.y));
      }
    __syncwarp();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (kLanes > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = top;
      __syncthreads();
      top = sh[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, sh[i]);
    }
    if (ln != 0) continue;
    if (ok) {
      offer((int)(lab >> p.shift), at_log);
      top = fmaxf(top, at_log + (float)exponent(p.fw[lab]));
    }
    // c = mant · 2^e; zeros, infinities and NaN are their own mant
    float mant = c;
    int e = 0;
    if (finite_bits(c) != 0) mant = frexpf(c, &e);
    // the row's largest |softmax − 1[label]| 2^{-kw}, below 2^floor(top) · 2; a finite factor, so that nothing is multiplied by an infinity
    int to = top > -1000.f ? (int)floorf(top < 1000.f ? top : 1000.f) - kScaleTop : -126;
    to = to < -126 ? -126 : to > 126 ? 126 : to;
    p.row_exp[row] = e + to;
    p.stat[row] = RowStat{a.x, rest, at_label, mant, mant * pow2i(-to), e + fx, {}};
  }
  __syncthreads();
  for (int t = threadIdx.x; t < kept; t += 256)
    if (mine[t] != kNoRow) atomicMax(p.largest + t, mine[t]);
}

// fp32 operands: kept exponentials of a row to G for gx, in place, and to G for gw, beside it.  kLanes threads a row; blockIdx.y
// shares the classes of a row where there are few rows.  Bound by memory: 12 bytes for each row and class, 1003 x 32,003 in 70 us
// (5.5 TB/s).  Two eights a thread at a time take twice the registers and 91 us; 48 registers 74, 40 registers 81.
template <int kLanes>
__global__ void __launch_bounds__(256, 4)
k_loss_grad(const __grid_constant__ JoinArgs p) {
  pdl_wait();
  const int ln = threadIdx.x % kLanes, row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (kLanes == 32 && row >= p.n) return;
  const float2* part = p.part + (int64_t)row * p.parts;
  const RowStat r = p.stat[row];
  const bool ok = has_class(p.y[row], p.V);
  const int64_t lab = ok ? p.y[row] - p.v0 : -1;
  uint16_t *g = p.g + (int64_t)row * p.ldg, *g2 = p.g2 + (int64_t)row * p.ldg;
  for (int col = (blockIdx.y * kLanes + ln) * 8; col < p.len; col += gridDim.y * kLanes * 8) {
    const uint4 h = *reinterpret_cast<const uint4*>(g + col), l = *reinterpret_cast<const uint4*>(g + p.plane + col);
    const float4 f0 = *reinterpret_cast<const float4*>(p.fw + p.v0 + col), f1 = *reinterpret_cast<const float4*>(p.fw + p.v0 + col + 4);
    const int t = (p.v0 + col) >> p.shift, to_w = r.to_w - part_scale(p.largest[t]);
    const float scale = ex2((part[t].x - r.top) - r.rest) * pow2i(-kExpScale), w = r.mant * pow2i(to_w < 126 ? to_w : 126);
    const int at = lab >= col && lab < col + 8 ? (int)(lab - col) : -1;
    const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {l.x, l.y, l.z, l.w};
    const float fs[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
    uint32_t o[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&hs[i])), v = __half22float2(*reinterpret_cast<const __half2*>(&ls[i]));
      const float a = at == 2 * i ? r.at_label : (u.x + v.x) * scale, b = at == 2 * i + 1 ? r.at_label : (u.y + v.y) * scale;
      const float ax = ok ? a * r.to_x * fs[2 * i] : 0.f, bx = ok ? b * r.to_x * fs[2 * i + 1] : 0.f, aw = ok ? a * w : 0.f, bw = ok ? b * w : 0.f;
      o[0][i] = pair16<kFmtPlanes>(ax, bx, false); o[1][i] = pair16<kFmtPlanes>(ax, bx, true);
      o[2][i] = pair16<kFmtPlanes>(aw, bw, false); o[3][i] = pair16<kFmtPlanes>(aw, bw, true);
    }
    *reinterpret_cast<uint4*>(g + col) = make_uint4(o[0][0], o[0][1], o[0][2], o[0][3]);
    *reinterpret_cast<uint4*>(g + p.plane + col) = make_uint4(o[1][0], o[1][1], o[1][2], o[1][3]);
    *reinterpret_cast<uint4*>(g2 + col) = make_uint4(o[2][0], o[2][1], o[2][2], o[2][3]);
    *reinterpret_cast<uint4*>(g2 + p.plane + col) = make_uint4(o[3][0], o[3][1], o[3][2], o[3][3]);
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

// where things lie in the workspace; everything is 256-byte aligned
struct LossPlan {
  int planes, pack_x, pack_w, parts, per_tile, keep, piece, together;
  int tiny, tiny_ld, tiny_ldg, tiny_smem;     // CTAs of k_loss_tiny, 0: the general way
  Tiling score, gx, gw;                       // gx, gw: of the kept classes, or of a piece
  int64_t dp, ldg, x_plane, w_plane, g_plane;
  int64_t scale, lse, target, x, w, part, g, gx_acc, gw_acc, total;
  int64_t fx, fw, widest, stat, row_exp, largest, g2;       // fp32
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
  p.scale = take(4);
  p.lse = take((int64_t)a.n * 4);
  p.target = take((int64_t)a.n * 4);
  p.x_plane = (int64_t)a.n * p.dp;
  if (p.pack_x || a.want_grad) p.x = take(p.x_plane * 2 * p.planes);
  p.w_plane = (int64_t)a.V * p.dp;
  if (p.pack_w) p.w = take(p.w_plane * 2 * p.planes);
  p.part = take((int64_t)p.parts * a.n * 8);
  if (p.planes == 2) {
    p.fx = take((int64_t)a.n * 4);
    p.fw = take(((int64_t)a.V + 256) * 4);          // a tile reads all of its columns' factors
    if (a.want_grad) {
      p.widest = take((int64_t)p.parts * a.n * 8);
      p.stat = take((int64_t)a.n * sizeof(RowStat));
      p.row_exp = take((int64_t)a.n * 4);
      p.largest = take((int64_t)p.parts * 4);
    }
  }
  if (a.want_grad) {
    int64_t len = ((int64_t)a.keep_mb << 20) / ((int64_t)a.n * (p.planes == 2 ? 8 : 2)) / 256 * 256;
    if (len < 256) len = 256;
    p.keep = p.piece = (int)(len < a.V ? len : a.V);
    p.ldg = ((int64_t)p.piece + 7) / 8 * 8;
    p.g_plane = (int64_t)a.n * p.ldg;
    p.g = take(p.g_plane * 2 * p.planes);
    if (p.planes == 2) p.g2 = take(p.g_plane * 4);
    const bool pieces = p.piece < a.V;
    p.gw = choose_tiling(1, p.piece, a.d, a.n, p.planes, false, pieces ? 1 : 16);
    p.gx = choose_tiling(1, a.n, a.d, p.piece, p.planes, false, pieces ? 1 : 64);
    // both in one launch where their tiles, of one kind, are one round: a launch less, and a third of the SMs does not wait
    if (a.want_gx && !pieces && (p.gw.kind == kOne128 || p.gw.kind == kOne64)) {
      const Tiling t = choose_tiling(1, a.n, a.d, p.piece, p.planes, false, 64, 1, p.gw.kind);
      auto tiles = [&](const Tiling& u, int64_t M) { return (M + 127) / 128 * ((a.d + tiling_cols(u.kind) - 1) / tiling_cols(u.kind)) * u.splits; };
      if ((p.gw.kb_split > t.kb_split ? p.gw.kb_split : t.kb_split) <= EpiGrad::kLongK / kG16K && tiles(p.gw, a.V) + tiles(t, a.n) <= 148) {
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
  int* found = reinterpret_cast<int*>(ws + p.scale);
  float *lse = reinterpret_cast<float*>(ws + p.lse), *target = reinterpret_cast<float*>(ws + p.target);
  uint16_t *xb = reinterpret_cast<uint16_t*>(ws + p.x), *wb = reinterpret_cast<uint16_t*>(ws + p.w), *gb = reinterpret_cast<uint16_t*>(ws + p.g);
  float2* part = reinterpret_cast<float2*>(ws + p.part);
  const bool f32 = p.planes == 2;
  float *fx = reinterpret_cast<float*>(ws + p.fx), *fw = reinterpret_cast<float*>(ws + p.fw);
  float2* widest = reinterpret_cast<float2*>(ws + p.widest);
  int *row_exp = reinterpret_cast<int*>(ws + p.row_exp), *largest = reinterpret_cast<int*>(ws + p.largest);
  uint16_t* g2 = reinterpret_cast<uint16_t*>(ws + p.g2);
  Chain chain{s};
  int r = 0;

  ScaleRef scale{a.dtype == kF16 ? 13 : 0, nullptr};       // without coefficients the largest is 1
  if (a.dtype == kF16 && a.coef != nullptr && a.want_grad) {
    scale.found = found;
    if ((r = chain.launch(k_loss_coef, dim3(1), 256, 0, 1, a.coef, a.y, a.n, a.V, found)) != 0) return r;
  }
  if (p.pack_x || p.pack_w) {
    const PackArgs px{a.x, a.n, a.ldx, xb, p.dp, p.x_plane}, pw{a.w, a.V, a.ldw, wb, p.dp, p.w_plane};
    if (f32) {
      // a warp takes a row up to 1024 columns, and the block one above
      const int64_t rows = (int64_t)a.n + a.V;
      auto planes = [&](auto kernel, int lanes) {
        return chain.launch(kernel, dim3(blocks_for(rows * lanes, 148 * 8)), 256, 0, 1, px, pw, a.d, a.y, a.n, a.V, fx, fw, largest,
                            a.want_grad ? p.parts : 0);
      };
      r = a.d <= 1024 ? planes(k_loss_planes<32>, 32) : planes(k_loss_planes<256>, 256);
    } else {
      const unsigned bx = p.pack_x ? blocks_for((int64_t)a.n * (p.dp / 8), 148 * 8) : 0, bw = p.pack_w ? blocks_for((int64_t)a.V * (p.dp / 8), 148 * 8) : 0;
      auto pack = [&](auto kernel) { return chain.launch(kernel, dim3(bx + bw), 256, 0, 1, px, pw, a.d, a.y, a.V, (int)bx); };
      r = a.dtype == kBF16 ? pack(k_loss_pack<__nv_bfloat16>) : pack(k_loss_pack<__half>);
    }
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
  es.part = part; es.target = target; es.y = a.y; es.n = a.n; es.V = a.V; es.parts = p.parts; es.per_tile = p.per_tile; es.keep = p.keep;
  es.fx = fx; es.fw = fw; es.widest = a.want_grad ? widest : nullptr;
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
  int64_t share = a.want_grad ? (148 * 6 + a.n - 1) / a.n : 1, most = ((int64_t)p.keep + 8191) / 8192;
  if (share > most) share = most < 1 ? 1 : most;
  const bool warp_rows = p.parts <= 64 && a.V <= 2048;      // a warp a row; with and without gradients alike, so that losses are the same
  const dim3 by_warps((unsigned)(a.n + 7) / 8), shared((unsigned)a.n, (unsigned)share);
  if (f32) {
    j.widest = widest; j.fx = fx; j.fw = fw; j.row_exp = row_exp; j.largest = largest; j.g2 = g2;
    if (a.want_grad) j.stat = reinterpret_cast<RowStat*>(ws + p.stat);
    auto join = [&](auto kernel, unsigned blocks) { return chain.launch(kernel, dim3(blocks < 148 * 4 ? blocks : 148 * 4), 256, 0, 1, j); };
    r = p.parts <= 256 ? join(k_loss_join<32>, by_warps.x) : join(k_loss_join<256>, (unsigned)a.n);
  } else {
    r = warp_rows ? chain.launch(k_loss_rows<32>, by_warps, 256, 0, 1, j) : chain.launch(k_loss_rows<256>, shared, 256, 0, 1, j);
  }
  if (r || !a.want_grad) return r;

  const Operand16 xz{xb, a.n, a.d, p.dp, p.x_plane, p.planes};      // rows without a class are zeros
  const int64_t es_out = a.dtype == kF32 ? 4 : 2;
  for (int v0 = 0; v0 < a.V; v0 += p.piece) {
    const int len = a.V - v0 < p.piece ? a.V - v0 : p.piece;
    const Operand16 gop{gb, a.n, len, p.ldg, p.g_plane, p.planes}, gop_w{f32 ? g2 : gb, a.n, len, p.ldg, p.g_plane, p.planes};
    Gemm16Args gs = g;
    gs.N = len; gs.b_n0 = v0;
    if (f32) {
      if (v0 > 0) {                            // beyond the kept classes: scores and exponentials once more
        EpiScore::Params again = es;
        if ((r = make_out_map(&again.e, gop, 0)) != 0) return r;
        again.part = nullptr; again.widest = nullptr; again.keep = len; again.v0 = v0;
        if ((r = product16<EpiScore>(chain, p.planes, p.score.kind, gs, x, w, again)) != 0) return r;
      }
      j.v0 = v0; j.len = len;
      r = warp_rows ? chain.launch(k_loss_grad<32>, by_warps, 256, 0, 1, j) : chain.launch(k_loss_grad<256>, shared, 256, 0, 1, j);
      if (r) return r;
    } else if (v0 > 0) {                       // scores once more
      EpiG::Params eg = {};
      if ((r = make_out_map(&eg.g, gop, a.dtype == kBF16)) != 0) return r;
      eg.lse = lse; eg.coef = a.coef; eg.y = a.y; eg.scale = scale; eg.n = a.n; eg.V = a.V; eg.len = len; eg.v0 = v0; eg.dtype = a.dtype;
      Launch16<EpiG, 1> l = {{gs}, {eg}};
      if ((r = launch_tiled<1, EpiG>(chain, choose_tiling(1, a.n, len, a.d, 1, false, 1).kind, l, x, w)) != 0) return r;
    }
    EpiGrad::Params e = {};
    e.scale = scale; e.dtype = a.dtype;
    Gradient q[2];
    // gw[v0.., :] = Gᵀ x
    q[0] = Gradient{g, gop_w, xz, e};
    q[0].g.M = len; q[0].g.N = a.d; q[0].g.K = a.n; q[0].g.a_mn = q[0].g.b_mn = 1;
    q[0].e.out = reinterpret_cast<uint8_t*>(a.gw) + (int64_t)v0 * a.d * es_out;
    q[0].e.exps = largest; q[0].e.exp_parts = 1; q[0].e.exp_first = v0; q[0].e.exp_shift = j.shift;
    if (p.gw.splits > 1) q[0].e.acc = reinterpret_cast<float*>(ws + p.gw_acc);
    if ((r = prepare(q[0], p.gw)) != 0) return r;
    if (!p.together && (r = gradient(chain, p.planes, p.gw.kind, q[0])) != 0) return r;
    if (a.gx == nullptr) continue;
    // gx += G w[v0.., :]
    q[1] = Gradient{g, gop, w, e};
    q[1].g.M = a.n; q[1].g.N = a.d; q[1].g.K = len; q[1].g.b_k0 = v0; q[1].g.b_mn = 1;
    q[1].e.out = a.gx; q[1].e.exps = row_exp;
    if (p.gx.splits > 1 || p.piece < a.V) q[1].e.acc = reinterpret_cast<float*>(ws + p.gx_acc);
    if (p.piece < a.V) { q[1].e.read = v0 > 0; q[1].e.write = v0 + len < a.V; }
    if ((r = prepare(q[1], p.gx)) != 0) return r;
    r = p.together ? gradients(chain, p.planes, p.gx.kind, q) : gradient(chain, p.planes, p.gx.kind, q[1]);
    if (r) return r;
  }
  return 0;
}

}  // extern "C"
