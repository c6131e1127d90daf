// Softmax cross entropy of rows over many classes, with its gradients, without keeping the scores.
//
//   s_ij = x_i · w_j        loss_i = c_i (log Σ_j e^{s_ij} − s_{i,y_i})        x [n, d], w [V, d], y_i in 0..V-1 or -1
//   G_ij = c_i (e^{s_ij − lse_i} − [j = y_i])        gx = G w        gw = Gᵀ x
//
// The scores are tiles of a product on the tensor cores (gemm16.cuh) and never leave the SM: its epilogue keeps each row's
// running maximum m and sum Σ e^{s−m} over the tile's classes, and the score of the row's label; a second, small kernel
// joins the tiles of a row.  The gradient takes the classes in pieces: the piece's scores are made again, turned into G
// (which is kept for one piece only, in the type of the operands) and multiplied with the piece of w and with x.  gw of a
// piece is complete, gx is summed over the pieces in fp32.  Sums have a fixed order: results do not vary from run to run.
//
// Scores, maxima, sums and losses are fp32 (in units of log2 e: 2^x is the hardware's exponential).  G is rounded to the
// operands' type: bf16 for bf16; fp16 for fp16, scaled by a power of two so that the largest coefficient is near 2^13;
// two planes of fp16 for fp32, where x and w are such planes too (22 bits).
#include "gemm16.cuh"

namespace psb {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// device scalars of a call: largest finite |x|, |w|, |c| as bits; then the exponents derived from them
struct LossScal {
  uint32_t max_x, max_w, max_c, pad;
};
// exponent that brings the largest finite magnitude into [2^top, 2^(top+1))
__device__ __forceinline__ int scale_exp(uint32_t bits, int top) {
  if (bits == 0) return 0;
  const int e = (int)(bits >> 23) - 127;             // subnormals count as 2^-127: the scale only has to be representable
  const int k = top - e;
  return k > 126 ? 126 : k;
}
__device__ __forceinline__ float pow2i(int e) {       // 2^e, kept finite and normal
  e = e > 127 ? 127 : e;
  return e < -126 ? 0.f : __int_as_float((e + 127) << 23);
}
struct Scales { int x, w, g; };
// fp32: planes use the whole range of fp16; 16-bit types are taken as they are, and fp16 gradients are scaled
__device__ __forceinline__ Scales scales_of(const LossScal* s, int dtype) {
  Scales k{0, 0, 0};
  if (dtype == kF32) { k.x = scale_exp(s->max_x, 14); k.w = scale_exp(s->max_w, 14); }
  if (dtype != kBF16) k.g = scale_exp(s->max_c, 13);
  return k;
}

// ------------------------------------------------------------------ preparation
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v) {
  __shared__ uint32_t sh[32];
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < (blockDim.x >> 5) ? sh[threadIdx.x] : 0u;
  if (threadIdx.x < 32) v = __reduce_max_sync(0xffffffffu, v);
  return v;
}
__device__ __forceinline__ bool has_class(int64_t y, int V) { return y >= 0 && y < V; }

// Labels as int32 (-1: none), coefficients (0 where there is no class), the largest coefficient.  A label outside the classes
// is recorded in the status word and counts as none.
__global__ void __launch_bounds__(256)
k_loss_labels(const int64_t* __restrict__ y, const float* __restrict__ coef, int n, int V, int* __restrict__ label, float* __restrict__ c,
              LossScal* scal, uint32_t* status) {
  uint32_t top = 0;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
    const int64_t v = y[i];
    const bool ok = has_class(v, V);
    if (v != -1 && !ok) set_status(status, kBadIndex, (uint32_t)i, (uint32_t)v);
    label[i] = ok ? (int)v : -1;
    const float cv = ok ? (coef != nullptr ? coef[i] : 1.f) : 0.f;
    c[i] = cv;
    top = max(top, finite_bits(cv));
  }
  top = block_max_u32(top);
  if (threadIdx.x == 0 && top != 0) atomicMax(&scal->max_c, top);
}

// Largest finite magnitude of fp32 rows; rows without a class do not count (y null: all rows do).
__global__ void __launch_bounds__(256)
k_loss_absmax(const float* __restrict__ a, int64_t rows, int cols, int64_t ld, const int64_t* __restrict__ y, int V, uint32_t* out) {
  uint32_t top = 0;
  const bool vec = ((reinterpret_cast<uintptr_t>(a) & 15) | (ld & 3)) == 0;
  const int per = (cols + 3) / 4;
  const int64_t total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
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
  top = block_max_u32(top);
  if (threadIdx.x == 0 && top != 0) atomicMax(out, top);
}

// Rows of any stride and alignment into operand planes [plane][row][ldo]; rows without a class become zeros, whatever they
// held (y null: none do).  which: 0 = x, 1 = w, the exponent that scales fp32.
template <typename T>
__global__ void __launch_bounds__(256)
k_loss_pack(const T* __restrict__ a, int64_t rows, int cols, int64_t ld, const int64_t* __restrict__ y, int V, uint16_t* __restrict__ out,
            int64_t ldo, int64_t plane, const LossScal* scal, int which) {
  const int per = (int)(ldo / 8);
  const int64_t total = rows * per;
  float s = 1.f;
  if (sizeof(T) == 4) {
    const Scales k = scales_of(scal, kF32);
    s = pow2i(which ? k.w : k.x);
  }
  const bool vec = ((reinterpret_cast<uintptr_t>(a) & 15) | ((ld * sizeof(T)) & 15)) == 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    const T* p = a + r * ld + c;
    const bool none = y != nullptr && !has_class(y[r], V);
    alignas(16) T v[8];
    if (none) {
      for (int j = 0; j < 8; ++j) v[j] = T(0);
    } else if (vec && c + 8 <= cols) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(v)[j] = reinterpret_cast<const uint4*>(p)[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? p[j] : T(0);
    }
    uint16_t* dst = out + r * ldo + c;
    if constexpr (sizeof(T) == 4) {
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __half h0, l0, h1, l1;
        split16((float)v[2 * j] * s, h0, l0);
        split16((float)v[2 * j + 1] * s, h1, l1);
        h[j] = pack_half2(h0, h1); l[j] = pack_half2(l0, l1);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(dst + plane) = make_uint4(l[0], l[1], l[2], l[3]);
    } else {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(v);
    }
  }
}

// ------------------------------------------------------------------ epilogues
// Each row's maximum and Σ 2^(s−m) over half a tile's classes, and the score of its label, in units of log2 e.
struct EpiScore {
  struct Params {
    float2* part;              // [2 · class tiles][n]
    float* target;             // [n]
    const int* label;
    const LossScal* scal;
    int n, V, dtype;
  };
  const Params& p;
  float scale, m, s;
  int row, lab;
  int64_t at;
  __device__ __forceinline__ EpiScore(const Params& p_, const Gemm16Args&, const Tile16& w, int row_, int half)
      : p(p_), m(-INFINITY), s(0.f), row(row_), lab(-2) {
    const Scales k = scales_of(p.scal, p.dtype);
    scale = kLog2e * pow2i(-(k.x + k.w));
    if (row < p.n) lab = p.label[row];
    at = (int64_t)(w.tn * 2 + half) * p.n + row;
  }
  __device__ __forceinline__ void chunk(float (&v)[32], int col) {
    if (col >= p.V) return;
    float top = -INFINITY;
    const int left = p.V - col;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] *= scale;
      if (left < 32) v[j] = j < left ? v[j] : -INFINITY;
    }
    if ((unsigned)(lab - col) < 32u) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) t = j == lab - col ? v[j] : t;
      p.target[row] = t;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j]);
    // without a finite score yet the reference is 0: 2^(-inf) is 0 and nothing is subtracted from an infinity
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) sum += ex2(v[j] - ref);
    s = s * ex2(m - ref) + sum;
    m = mn;
  }
  __device__ __forceinline__ void end() {
    if (row < p.n) p.part[at] = make_float2(m, s);
  }
};

// G of a piece of the classes, in the operands' type
struct EpiG {
  struct Params {
    uint16_t* out;             // [plane][n][ldg]
    int64_t ldg, plane;
    const float* lse;          // [n], log2
    const float* c;
    const int* label;
    const LossScal* scal;
    int n, len, v0, dtype;
  };
  const Params& p;
  float scale, c, lse;
  int row, lab;
  __device__ __forceinline__ EpiG(const Params& p_, const Gemm16Args&, const Tile16&, int row_, int)
      : p(p_), c(0.f), lse(0.f), row(row_), lab(-1) {
    const Scales k = scales_of(p.scal, p.dtype);
    scale = kLog2e * pow2i(-(k.x + k.w));
    if (row < p.n) {
      lab = p.label[row];
      lse = p.lse[row];
      c = lab >= 0 ? p.c[row] * pow2i(k.g) : 0.f;
      lab = lab >= 0 ? lab - p.v0 : -1;
      if (lab < 0 && p.label[row] >= 0) lab = -2;         // the row's class lies in another piece
    }
  }
  __device__ __forceinline__ void chunk(float (&v)[32], int col) {
    if (row >= p.n || col >= p.ldg) return;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = ex2(v[j] * scale - lse);
      v[j] = lab == -1 ? 0.f : c * (v[j] - (j == lab - col ? 1.f : 0.f));
    }
    uint16_t* dst = p.out + (int64_t)row * p.ldg + col;
    const int left = (int)p.ldg - col;                     // a multiple of 8; what lies behind the piece is not read
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      if (j >= left) break;
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = v[j + 2 * i], b = v[j + 2 * i + 1];
        if (p.dtype == kBF16) {
          const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
          h[i] = *reinterpret_cast<const uint32_t*>(&t);
        } else {
          __half h0, l0, h1, l1;
          split16(a, h0, l0);
          split16(b, h1, l1);
          h[i] = pack_half2(h0, h1);
          l[i] = pack_half2(l0, l1);
        }
      }
      *reinterpret_cast<uint4*>(dst + j) = make_uint4(h[0], h[1], h[2], h[3]);
      if (p.dtype == kF32) *reinterpret_cast<uint4*>(dst + p.plane + j) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  }
  __device__ __forceinline__ void end() {}
};

__device__ __forceinline__ void store_as(void* out, int64_t at, float v, int dtype) {
  if (dtype == kF32) reinterpret_cast<float*>(out)[at] = v;
  else if (dtype == kBF16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
}
// 1 / (scale of G times scale of the other operand)
__device__ __forceinline__ float grad_scale(const LossScal* scal, int dtype, int with_w) {
  const Scales k = scales_of(scal, dtype);
  return pow2i(-(k.g + (with_w ? k.w : k.x)));
}

// A gradient: to the result, or raw fp32 sums to `acc` (piece by piece, or one slot per split of K)
struct EpiGrad {
  struct Params {
    void* out;
    float* acc;
    int64_t ldo, slot;
    const LossScal* scal;
    int M, N, dtype, with_w;
    int read, write;           // acc is added to the product; the sum goes to acc instead of the result
  };
  const Params& p;
  float scale;
  int row;
  float* acc;
  __device__ __forceinline__ EpiGrad(const Params& p_, const Gemm16Args&, const Tile16& w, int row_, int)
      : p(p_), row(row_) {
    scale = grad_scale(p.scal, p.dtype, p.with_w);
    acc = p.acc != nullptr ? p.acc + w.split * p.slot + (int64_t)row * p.N : nullptr;
  }
  __device__ __forceinline__ void chunk(float (&v)[32], int col) {
    if (row >= p.M || col >= p.N) return;
    const int left = p.N - col;
    const bool vec = left >= 32 && (p.N & 3) == 0;         // acc is 16-byte aligned and its rows are N floats
    if (p.read) {
      if (vec) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 t = *reinterpret_cast<const float4*>(acc + col + j);
          v[j] += t.x; v[j + 1] += t.y; v[j + 2] += t.z; v[j + 3] += t.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) if (j < left) v[j] += acc[col + j];
      }
    }
    if (p.write) {
      if (vec) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(acc + col + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) if (j < left) acc[col + j] = v[j];
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= scale;
    const int64_t at = (int64_t)row * p.ldo + col;
    if (left >= 32 && p.dtype == kF32 && ((reinterpret_cast<uintptr_t>(p.out) & 15) | (p.ldo & 3)) == 0) {
      float* dst = reinterpret_cast<float*>(p.out) + at;
#pragma unroll
      for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(dst + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else if (left >= 32 && p.dtype != kF32 && ((reinterpret_cast<uintptr_t>(p.out) & 15) | (p.ldo & 7)) == 0) {
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + at;
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p.dtype == kBF16) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[j + 2 * i], v[j + 2 * i + 1]);
            h[i] = *reinterpret_cast<const uint32_t*>(&t);
          } else {
            h[i] = pack_half2(__float2half_rn(v[j + 2 * i]), __float2half_rn(v[j + 2 * i + 1]));
          }
        }
        *reinterpret_cast<uint4*>(dst + j) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) if (j < left) store_as(p.out, at + j, v[j], p.dtype);
    }
  }
  __device__ __forceinline__ void end() {}
};

// ------------------------------------------------------------------ joining
// The halves of a row's tiles to its log-sum-exp (log2) and its loss.  kRows rows a block, the rest of its threads share
// the tiles of a row.
template <int kRows>
__global__ void __launch_bounds__(256)
k_loss_join(const float2* __restrict__ part, int parts, int n, const float* __restrict__ target, const int* __restrict__ label,
            const float* __restrict__ c, float* __restrict__ lse, float* __restrict__ loss) {
  constexpr int kLanes = 256 / kRows;
  __shared__ float2 sh[kLanes][kRows];
  const int rr = threadIdx.x % kRows, ln = threadIdx.x / kRows, row = blockIdx.x * kRows + rr;
  float m = -INFINITY, s = 0.f;
  if (row < n)
    for (int q = ln; q < parts; q += kLanes) {
      const float2 v = part[(int64_t)q * n + row];
      const float mn = fmaxf(m, v.x), ref = mn == -INFINITY ? 0.f : mn;
      s = s * ex2(m - ref) + v.y * ex2(v.x - ref);
      m = mn;
    }
  sh[ln][rr] = make_float2(m, s);
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (ln < o) {
      const float2 a = sh[ln][rr], b = sh[ln + o][rr];
      const float mn = fmaxf(a.x, b.x), ref = mn == -INFINITY ? 0.f : mn;
      sh[ln][rr] = make_float2(mn, a.y * ex2(a.x - ref) + b.y * ex2(b.x - ref));
    }
  }
  if (ln == 0 && row < n) {
    const float2 v = sh[0][rr];
    const float l2 = log2f(v.y);
    lse[row] = v.x + l2;
    loss[row] = label[row] >= 0 ? c[row] * (kLn2 * ((v.x - target[row]) + l2)) : 0.f;
  }
}

// the splits of K to the result
__global__ void __launch_bounds__(256)
k_loss_sum(const float* __restrict__ acc, int splits, int64_t slot, int64_t numel, void* out, const LossScal* scal, int dtype, int with_w) {
  const float scale = grad_scale(scal, dtype, with_w);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < numel; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int q = 0; q < splits; ++q) v += acc[q * slot + i];
    store_as(out, i, v * scale, dtype);
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
  int n, V, d, dtype, want_grad, pad;
  void* ws;
  int64_t ws_bytes;
  uint32_t* status;
};

}  // namespace psb

using namespace psb;

namespace {

// where things lie in the workspace; everything is 256-byte aligned
struct LossPlan {
  int planes, pack_w, piece, tile;            // tile: 0 = pairs 256x256, 1 = 128x128, 2 = 128x64, of the scores
  int parts, gx_splits, gw_splits;
  int64_t dp, ldg, x_plane, w_plane, g_plane;
  int64_t scal, label, c, lse, target, x, w, part, g, gx_acc, gw_acc, total;
};

constexpr int64_t kPieceBytes = (int64_t)256 << 20;    // of G

int tile_kind(int64_t M, int64_t N) {
  // 256x256 tiles of pairs from 48 tiles on (two thirds of the pairs of SMs); below, 128x128 tiles, or 128x64 where
  // those would leave more than half of the SMs idle
  if (((M + 255) / 256) * ((N + 255) / 256) >= 48) return 0;
  return ((M + 127) / 128) * ((N + 127) / 128) >= 74 ? 1 : 2;
}
int tile_cols(int kind) { return kind == 0 ? 256 : kind == 1 ? 128 : 64; }
int64_t tiles_of(int kind, int64_t M, int64_t N) {
  const int64_t m = kind == 0 ? 256 : 128, c = tile_cols(kind);
  return ((M + m - 1) / m) * ((N + c - 1) / c);
}
// K in so many pieces that the SMs are busy, eight blocks of 64 a piece at least; pieces' sums are stored and added up
int split_count(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = tiles_of(tile_kind(M, N), M, N), nkb = (K + kG16K - 1) / kG16K;
  int64_t s = 148 / (tiles < 1 ? 1 : tiles);
  if (s > nkb / 8) s = nkb / 8;
  if (s < 2) return 1;
  const int64_t per = (nkb + s - 1) / s;
  return (int)((nkb + per - 1) / per);
}

LossPlan loss_plan(const LossArgs& a) {
  LossPlan p = {};
  p.planes = a.dtype == kF32 ? 2 : 1;
  p.dp = (a.d + 7) / 8 * 8;
  p.pack_w = p.planes == 2 || (a.ldw & 7) || (reinterpret_cast<uintptr_t>(a.w) & 15) || a.ldw < a.d;
  p.tile = tile_kind(a.n, a.V);
  p.parts = 2 * (int)((a.V + tile_cols(p.tile) - 1) / tile_cols(p.tile));
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  p.scal = take(sizeof(LossScal));
  p.label = take((int64_t)a.n * 4);
  p.c = take((int64_t)a.n * 4);
  p.lse = take((int64_t)a.n * 4);
  p.target = take((int64_t)a.n * 4);
  p.x_plane = (int64_t)a.n * p.dp;
  p.x = take(p.x_plane * 2 * p.planes);
  p.w_plane = (int64_t)a.V * p.dp;
  if (p.pack_w) p.w = take(p.w_plane * 2 * p.planes);
  p.part = take((int64_t)p.parts * a.n * 8);
  if (a.want_grad) {
    int64_t len = kPieceBytes / ((int64_t)a.n * 2 * p.planes) / 256 * 256;
    if (len < 256) len = 256;
    p.piece = (int)(len < a.V ? len : a.V);
    p.ldg = (p.piece + 7) / 8 * 8;
    p.g_plane = (int64_t)a.n * p.ldg;
    p.g = take(p.g_plane * 2 * p.planes);
    p.gx_splits = p.piece >= a.V ? split_count(a.n, a.d, a.V) : 1;
    p.gw_splits = p.piece >= a.V ? split_count(a.V, a.d, a.n) : 1;
    if (a.gx != nullptr && (p.gx_splits > 1 || p.piece < a.V)) p.gx_acc = take((int64_t)p.gx_splits * a.n * a.d * 4);
    if (p.gw_splits > 1) p.gw_acc = take((int64_t)p.gw_splits * a.V * a.d * 4);
  }
  p.total = at;
  return p;
}

template <int kPlanes, bool kAMN, bool kBMN, class Epi>
int by_tile(int kind, const Gemm16Args& g, const Operand16& a, const Operand16& b, const typename Epi::Params& ep, cudaStream_t s) {
  if (kind == 0) return launch16<Cfg16<2, 256, kPlanes, kAMN, kBMN>, Epi>(g, a, b, ep, s);
  if (kind == 1) return launch16<Cfg16<1, 128, kPlanes, kAMN, kBMN>, Epi>(g, a, b, ep, s);
  return launch16<Cfg16<1, 64, kPlanes, kAMN, kBMN>, Epi>(g, a, b, ep, s);
}
template <bool kAMN, bool kBMN, class Epi>
int by_planes(int planes, int kind, const Gemm16Args& g, const Operand16& a, const Operand16& b, const typename Epi::Params& ep, cudaStream_t s) {
  return planes == 2 ? by_tile<2, kAMN, kBMN, Epi>(kind, g, a, b, ep, s) : by_tile<1, kAMN, kBMN, Epi>(kind, g, a, b, ep, s);
}

unsigned blocks_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 148 * 8 ? 148 * 8 : b);
}
template <typename T>
void pack(const void* a, int64_t rows, int cols, int64_t ld, const int64_t* y, int V, uint16_t* out, int64_t ldo, int64_t plane,
          const LossScal* scal, int which, cudaStream_t s) {
  k_loss_pack<T><<<blocks_for(rows * (ldo / 8)), 256, 0, s>>>(reinterpret_cast<const T*>(a), rows, cols, ld, y, V, out, ldo, plane, scal, which);
}
void pack_any(int dtype, const void* a, int64_t rows, int cols, int64_t ld, const int64_t* y, int V, uint16_t* out, int64_t ldo, int64_t plane,
              const LossScal* scal, int which, cudaStream_t s) {
  if (dtype == kF32) pack<float>(a, rows, cols, ld, y, V, out, ldo, plane, scal, which, s);
  else if (dtype == kBF16) pack<__nv_bfloat16>(a, rows, cols, ld, y, V, out, ldo, plane, scal, which, s);
  else pack<__half>(a, rows, cols, ld, y, V, out, ldo, plane, scal, which, s);
}

bool loss_args_ok(const LossArgs& a) {
  return a.n > 0 && a.V > 0 && a.d > 0 && a.dtype >= kF32 && a.dtype <= kF16 && a.V <= (1 << 30) && a.n <= (1 << 30) && a.d <= (1 << 30);
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
  if (p.total > a.ws_bytes || (reinterpret_cast<uintptr_t>(a.ws) & 255)) return (int)cudaErrorInvalidValue;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.ws);
  LossScal* scal = reinterpret_cast<LossScal*>(ws + p.scal);
  int* label = reinterpret_cast<int*>(ws + p.label);
  float *c = reinterpret_cast<float*>(ws + p.c), *lse = reinterpret_cast<float*>(ws + p.lse), *target = reinterpret_cast<float*>(ws + p.target);
  uint16_t *xb = reinterpret_cast<uint16_t*>(ws + p.x), *wb = reinterpret_cast<uint16_t*>(ws + p.w), *gb = reinterpret_cast<uint16_t*>(ws + p.g);
  float2* part = reinterpret_cast<float2*>(ws + p.part);
  const int bf16 = a.dtype == kBF16;

  cudaError_t e = cudaMemsetAsync(scal, 0, sizeof(LossScal), s);
  if (e != cudaSuccess) return (int)e;
  k_loss_labels<<<blocks_for(a.n), 256, 0, s>>>(a.y, a.coef, a.n, a.V, label, c, scal, a.status);
  if (a.dtype == kF32) {
    k_loss_absmax<<<blocks_for((int64_t)a.n * ((a.d + 3) / 4)), 256, 0, s>>>((const float*)a.x, a.n, a.d, a.ldx, a.y, a.V, &scal->max_x);
    k_loss_absmax<<<blocks_for((int64_t)a.V * ((a.d + 3) / 4)), 256, 0, s>>>((const float*)a.w, a.V, a.d, a.ldw, nullptr, a.V, &scal->max_w);
  }
  pack_any(a.dtype, a.x, a.n, a.d, a.ldx, a.y, a.V, xb, p.dp, p.x_plane, scal, 0, s);
  if (p.pack_w) pack_any(a.dtype, a.w, a.V, a.d, a.ldw, nullptr, a.V, wb, p.dp, p.w_plane, scal, 1, s);
  if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;

  const Operand16 x{xb, a.n, a.d, p.dp, p.x_plane, p.planes};
  const Operand16 w = p.pack_w ? Operand16{wb, a.V, a.d, p.dp, p.w_plane, p.planes} : Operand16{a.w, a.V, a.d, a.ldw, 0, 1};
  Gemm16Args g = {};
  g.batch = 1; g.splits = 1; g.bf16 = bf16; g.status = a.status;
  g.M = a.n; g.N = a.V; g.K = a.d;
  g.kb_split = (a.d + kG16K - 1) / kG16K;
  int r = by_planes<false, false, EpiScore>(p.planes, p.tile, g, x, w, EpiScore::Params{part, target, label, scal, a.n, a.V, a.dtype}, s);
  if (r) return r;
  if (a.n >= 256) k_loss_join<32><<<(a.n + 31) / 32, 256, 0, s>>>(part, p.parts, a.n, target, label, c, lse, a.loss);
  else k_loss_join<1><<<a.n, 256, 0, s>>>(part, p.parts, a.n, target, label, c, lse, a.loss);
  if ((e = cudaGetLastError()) != cudaSuccess || !a.want_grad) return (int)e;

  for (int v0 = 0; v0 < a.V; v0 += p.piece) {
    const int len = a.V - v0 < p.piece ? a.V - v0 : p.piece;
    const Operand16 gop{gb, a.n, len, p.ldg, p.g_plane, p.planes};
    Gemm16Args gs = g;
    gs.N = len; gs.b_n0 = v0;
    r = by_planes<false, false, EpiG>(p.planes, tile_kind(a.n, len), gs, x, w,
                                      EpiG::Params{gb, p.ldg, p.g_plane, lse, c, label, scal, a.n, len, v0, a.dtype}, s);
    if (r) return r;
    // gw[v0.., :] = Gᵀ x
    Gemm16Args gg = g;
    const int nkb = (a.n + kG16K - 1) / kG16K;
    gg.M = len; gg.N = a.d; gg.K = a.n; gg.splits = p.gw_splits; gg.kb_split = (nkb + p.gw_splits - 1) / p.gw_splits;
    const int64_t es = a.dtype == kF32 ? 4 : 2;
    EpiGrad::Params eg = {};
    eg.out = reinterpret_cast<uint8_t*>(a.gw) + (int64_t)v0 * a.d * es;
    eg.ldo = a.d; eg.scal = scal; eg.M = len; eg.N = a.d; eg.dtype = a.dtype; eg.with_w = 0;
    if (p.gw_splits > 1) { eg.acc = reinterpret_cast<float*>(ws + p.gw_acc); eg.slot = (int64_t)a.V * a.d; eg.write = 1; }
    r = by_planes<true, true, EpiGrad>(p.planes, tile_kind(len, a.d), gg, gop, x, eg, s);
    if (r) return r;
    if (p.gw_splits > 1)
      k_loss_sum<<<blocks_for((int64_t)a.V * a.d), 256, 0, s>>>(eg.acc, p.gw_splits, eg.slot, (int64_t)a.V * a.d, a.gw, scal, a.dtype, 0);
    if (a.gx == nullptr) continue;
    // gx += G w[v0.., :]
    Gemm16Args gx = g;
    const int vkb = (len + kG16K - 1) / kG16K;
    gx.M = a.n; gx.N = a.d; gx.K = len; gx.b_k0 = v0; gx.splits = p.gx_splits; gx.kb_split = (vkb + p.gx_splits - 1) / p.gx_splits;
    EpiGrad::Params ex = {};
    ex.out = a.gx; ex.ldo = a.d; ex.scal = scal; ex.M = a.n; ex.N = a.d; ex.dtype = a.dtype; ex.with_w = 1;
    const bool pieces = p.piece < a.V, last = v0 + len >= a.V;
    if (pieces || p.gx_splits > 1) {
      ex.acc = reinterpret_cast<float*>(ws + p.gx_acc);
      ex.slot = (int64_t)a.n * a.d;
      ex.read = v0 > 0;
      ex.write = p.gx_splits > 1 || !last;
    }
    r = by_planes<false, true, EpiGrad>(p.planes, tile_kind(a.n, a.d), gx, gop, w, ex, s);
    if (r) return r;
    if (p.gx_splits > 1)
      k_loss_sum<<<blocks_for((int64_t)a.n * a.d), 256, 0, s>>>(ex.acc, p.gx_splits, ex.slot, (int64_t)a.n * a.d, a.gx, scal, a.dtype, 1);
    if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
  }
  return 0;
}

}  // extern "C"
