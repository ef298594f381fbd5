// A gated layer and its gradient.  With g = x Wg^T, u = x Wu^T (weights [hidden][dim]),
//   out = act(g) u,  silu(g) = g / (1 + e^-g),  gelu(g) = g Phi(g);
//   dg = grad u act'(g),  du = grad act(g),  grad_x = dg Wg + du Wu,  grad_Wg = dg^T x,  grad_Wu = du^T x.
// Products by matrix instructions, their sums in 32 bits.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "checkpoint.h"
#include "operators_device.h"

namespace arb {
namespace {

typedef float F4 __attribute__((ext_vector_type(4)));

// 16 bytes of an operand: what a lane gives to a product.
template <typename T>
struct alignas(16) Chunk {
  T v[16 / sizeof(T)];
};

// acc[r] += sum over k of a(row 4 (lane / 16) + r, k) b(row lane % 16, k); a lane's chunk is its row lane % 16 at the
// k's number lane / 16 of as many.
__device__ __forceinline__ F4 Product(const Chunk<__bf16> &a, const Chunk<__bf16> &b, F4 acc) {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), acc, 0, 0, 0);
}
__device__ __forceinline__ F4 Product(const Chunk<_Float16> &a, const Chunk<_Float16> &b, F4 acc) {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), acc, 0, 0, 0);
}
__device__ __forceinline__ F4 Product(const Chunk<float> &a, const Chunk<float> &b, F4 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
  return acc;
}

// ------------------------------------------------------------------ activations

__device__ __forceinline__ float Sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

template <int kAct>
__device__ __forceinline__ float Act(float g) {
  if (kAct == kSilu) return g * Sigmoid(g);
  return 0.5f * g * erfcf(-0.70710678118654752f * g);
}

// act(g) and act'(g)
template <int kAct>
__device__ __forceinline__ void ActAndSlope(float g, float *act, float *slope) {
  if (kAct == kSilu) {
    const float s = Sigmoid(g);
    *act = g * s;
    *slope = s + *act * (1.0f - s);
  } else {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * g);
    *act = g * phi;
    *slope = phi + g * (0.39894228040143268f * expf(-0.5f * g * g));
  }
}

// ------------------------------------------------------------------ matrix products

constexpr int kTile = 128;      // rows and columns of a workgroup's tile
constexpr int kTileBytes = 128; // of k's along a row of a tile in the LDS
constexpr int kThreads = 256;
constexpr int kHalf = kTile / 2;  // hidden columns of a forward tile: as many of the gate, as many of up

// C[i][j] = sum over segments and k of A(i, k) B(j, k); a batch of two such products.
// An operand lies row by row with its k's side by side, or (ACROSS) k by k with its rows side by side.
struct Operand {
  const void *at[2];  // of each segment, or of each member of the batch
  long long stride;   // between rows, or between k's
};
struct Products {
  Operand a, b;
  long long rows;  // of A
  int columns;     // of C: rows of B
  long long inner;  // k's of a segment
  int segments;    // 1, or 2: C sums over both
  int batch;       // 1, or 2
  void *c[2];
  long long c_stride;
  // the k's of a tile shared out
  int splits;
  long long split_blocks;  // blocks of k's of each
  float *partial;          // [batch][splits][rows][columns] where there are several
};

// The chunk at (line, chunk) of a tile in the LDS: the order of the chunks of a line changes from line to line, so that the
// lanes of a product, who read one chunk of 16 lines, meet other banks.
template <typename T>
__device__ __forceinline__ Chunk<T> *ChunkAt(unsigned char *tile, int line, int chunk) {
  return reinterpret_cast<Chunk<T> *>(tile + line * kTileBytes + (((chunk ^ line) & 7) * 16));
}

// A tile's part of an operand on its way from memory to the LDS: kTile lines of kTileBytes.  What is beyond the operand is 0.
template <typename T, bool kAcross>
struct Stage {
  static constexpr int kVec = 16 / sizeof(T), kK = kTileBytes / sizeof(T), kPieces = kTile * 8 / kThreads;
  Chunk<T> piece[kPieces];

  // line(l): pointer to line l, its row beyond the operand: null; `lines`: of an ACROSS operand, lines from `first` on
  template <typename Line>
  __device__ __forceinline__ void Load(const Line &line, const T *base, long long stride, long long first, long long lines, long long k0, long long inner) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int q = p * kThreads + threadIdx.x;
      const T *from;
      long long left;
      if (!kAcross) {
        const long long k = k0 + q % 8 * kVec;
        const T *row = line(q / 8);
        from = row + k;
        left = row == nullptr ? 0 : inner - k;
      } else {
        const long long k = k0 + q / (kTile / kVec), m = first + q % (kTile / kVec) * kVec;
        from = base + k * stride + m;
        left = k < inner ? lines - m : 0;
      }
      if (left >= kVec) {
        const Pack<T, kVec> w = *reinterpret_cast<const Pack<T, kVec> *>(from);
#pragma unroll
        for (int c = 0; c < kVec; ++c) piece[p].v[c] = w.v[c];
      } else {
#pragma unroll
        for (int c = 0; c < kVec; ++c) piece[p].v[c] = c < left ? from[c] : T(0);
      }
    }
  }
  __device__ __forceinline__ void Store(unsigned char *tile) const {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int q = p * kThreads + threadIdx.x;
      if (!kAcross) {
        *ChunkAt<T>(tile, q / 8, q % 8) = piece[p];
      } else {
        const int k = q / (kTile / kVec), m = q % (kTile / kVec) * kVec;
#pragma unroll
        for (int c = 0; c < kVec; ++c) ChunkAt<T>(tile, m + c, k / kVec)->v[k % kVec] = piece[p].v[c];
      }
    }
  }
};

// A wave's 32 rows by all 128 columns: two by eight fragments of 16 x 16.
struct Tile {
  F4 acc[2][8];
  __device__ __forceinline__ void Clear() {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = F4{0, 0, 0, 0};
  }
  template <typename T>
  __device__ __forceinline__ void Add(unsigned char *a, unsigned char *b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Chunk<T> x[2], y[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = *ChunkAt<T>(a, wave * 32 + i * 16 + lane % 16, half * 4 + lane / 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = *ChunkAt<T>(b, j * 16 + lane % 16, half * 4 + lane / 16);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = Product(y[j], x[i], acc[i][j]);
    }
  }
};

// Four elements of a row from column `at` on, of `columns`.
template <typename T>
__device__ __forceinline__ void StoreFour(T *row, long long at, long long columns, const T (&v)[4]) {
  if (at + 4 <= columns) {
    *reinterpret_cast<Pack<T, 4> *>(row + at) = Pack<T, 4>{{v[0], v[1], v[2], v[3]}};
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (at + r < columns) row[at + r] = v[r];
  }
}

struct Forward {
  const void *x, *w_gate, *w_up;
  long long rows;
  int dim, hidden;
  long long x_stride, w_stride;
  void *out;
  long long out_stride;
  void *gate, *up;
  float *gate_scales, *up_scales;
  long long kept_stride;
};

// What a lane holds of four values in each of four fragments along a row: 16 of a group of 64, the other lanes of its
// row the rest.
template <typename T>
__device__ __forceinline__ void Keep(void *kept, float *scales, long long stride, long long row, int at, int hidden, const F4 *v) {
  const int quarter = (threadIdx.x & 63) / 16;
  if (scales == nullptr) {
    T *to = static_cast<T *>(kept) + row * stride;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T four[4] = {Round<T>(v[j][0]), Round<T>(v[j][1]), Round<T>(v[j][2]), Round<T>(v[j][3])};
      StoreFour<T>(to, at + j * 16 + quarter * 4, hidden, four);
    }
    return;
  }
  float most = 0.0f;  // (columns beyond the layer hold 0)
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) most = Larger(most, fabsf(v[j][r]));
  most = Larger(most, __shfl_xor(most, 16));
  most = Larger(most, __shfl_xor(most, 32));
  const float scale = ScaleOf(most);
  if (quarter == 0) scales[row * ((hidden + kScaleGroup - 1) / kScaleGroup) + at / kScaleGroup] = scale;
  signed char *to = static_cast<signed char *>(kept) + row * stride;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float four[4] = {v[j][0], v[j][1], v[j][2], v[j][3]};
    const Pack<signed char, 4> codes = CodesOf(four, scale);
    StoreFour<signed char>(to, at + j * 16 + quarter * 4, hidden, codes.v);
  }
}

static_assert(kHalf == kScaleGroup, "a wave holds whole groups");

template <typename T, int kAct>
__global__ void __launch_bounds__(kThreads) k_gated(const Forward a, long long tiles, int columns) {
  __shared__ __align__(16) unsigned char s_x[kTile * kTileBytes], s_w[kTile * kTileBytes];
  constexpr int kK = kTileBytes / sizeof(T);
  const T *x = static_cast<const T *>(a.x), *w_gate = static_cast<const T *>(a.w_gate), *w_up = static_cast<const T *>(a.w_up);
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long i0 = tile / columns * kTile;
    const int h0 = (int)(tile % columns) * kHalf;
    const auto x_line = [&](int l) { return i0 + l < a.rows ? x + (i0 + l) * a.x_stride : nullptr; };
    const auto w_line = [&](int l) {
      const int h = h0 + l % kHalf;
      return h < a.hidden ? (l < kHalf ? w_gate : w_up) + h * a.w_stride : nullptr;
    };
    Tile t;
    t.Clear();
    Stage<T, false> xs, ws;
    for (long long k0 = 0; k0 < a.dim; k0 += kK) {
      xs.Load(x_line, x, 0, 0, 0, k0, a.dim);
      ws.Load(w_line, x, 0, 0, 0, k0, a.dim);
      __syncthreads();
      xs.Store(s_x);
      ws.Store(s_w);
      __syncthreads();
      t.Add<T>(s_x, s_w);
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long row = i0 + wave * 32 + i * 16 + lane % 16;
      if (row >= a.rows) continue;  // (all four lanes of a row)
      T *out = static_cast<T *>(a.out) + row * a.out_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        T four[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) four[r] = Round<T>(Act<kAct>(t.acc[i][j][r]) * t.acc[i][j + 4][r]);
        StoreFour<T>(out, h0 + j * 16 + lane / 16 * 4, a.hidden, four);
      }
      if (a.gate != nullptr) {
        Keep<T>(a.gate, a.gate_scales, a.kept_stride, row, h0, a.hidden, t.acc[i]);
        Keep<T>(a.up, a.up_scales, a.kept_stride, row, h0, a.hidden, t.acc[i] + 4);
      }
    }
  }
}

template <typename T, bool kAcrossA, bool kAcrossB>
__global__ void __launch_bounds__(kThreads) k_products(const Products p, long long tiles, int columns, long long tiles_each) {
  __shared__ __align__(16) unsigned char s_a[kTile * kTileBytes], s_b[kTile * kTileBytes];
  constexpr int kK = kTileBytes / sizeof(T);
  const long long blocks = (p.inner + kK - 1) / kK;  // of a segment
  for (long long item = blockIdx.x; item < tiles; item += gridDim.x) {
    const long long one = item / tiles_each, tile = item % tiles_each;
    const int member = (int)(one / p.splits), split = (int)(one % p.splits);
    const long long i0 = tile / columns * kTile;
    const int j0 = (int)(tile % columns) * kTile;
    Tile t;
    t.Clear();
    Stage<T, kAcrossA> as;
    Stage<T, kAcrossB> bs;
    const long long end = min((split + 1) * p.split_blocks, blocks * p.segments);
    for (long long block = split * p.split_blocks; block < end; ++block) {
      const int segment = block >= blocks;
      const long long k0 = (block - segment * blocks) * kK;
      const T *a = static_cast<const T *>(p.a.at[member + segment]), *b = static_cast<const T *>(p.b.at[member + segment]);
      as.Load([&](int l) { return i0 + l < p.rows ? a + (i0 + l) * p.a.stride : nullptr; }, a, p.a.stride, i0, p.rows, k0, p.inner);
      bs.Load([&](int l) { return j0 + l < p.columns ? b + (j0 + l) * p.b.stride : nullptr; }, b, p.b.stride, j0, p.columns, k0, p.inner);
      __syncthreads();
      as.Store(s_a);
      bs.Store(s_b);
      __syncthreads();
      t.Add<T>(s_a, s_b);
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long row = i0 + wave * 32 + i * 16 + lane % 16;
      if (row >= p.rows) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = j0 + j * 16 + lane / 16 * 4;
        if (p.splits > 1) {
          const float four[4] = {t.acc[i][j][0], t.acc[i][j][1], t.acc[i][j][2], t.acc[i][j][3]};
          StoreFour<float>(p.partial + (one * p.rows + row) * p.columns, at, p.columns, four);
        } else {
          const T four[4] = {Round<T>(t.acc[i][j][0]), Round<T>(t.acc[i][j][1]), Round<T>(t.acc[i][j][2]), Round<T>(t.acc[i][j][3])};
          StoreFour<T>(static_cast<T *>(p.c[member]) + row * p.c_stride, at, p.columns, four);
        }
      }
    }
  }
}

// The sums of what was shared out, in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_products_join(const Products p) {
  const long long each = p.rows * p.columns, all = each * p.batch;
  for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < all; e += (long long)gridDim.x * kThreads) {
    const long long member = e / each, at = e - member * each, row = at / p.columns;
    const float *from = p.partial + member * p.splits * each + at;
    float sum = from[0];
    for (int s = 1; s < p.splits; ++s) sum += from[s * each];
    static_cast<T *>(p.c[member])[row * p.c_stride + (at - row * p.columns)] = Round<T>(sum);
  }
}

// ------------------------------------------------------------------ the layer's own gradient

struct Slopes {
  const void *grad_out;
  long long grad_out_stride;
  const void *gate, *up;
  const float *gate_scales, *up_scales;
  long long kept_stride;
  void *d_gate, *d_up;  // [rows][d_stride]
  long long d_stride, rows;
  int hidden;
};

constexpr int kSlopeVec = 4;

// d_gate and d_up, rounded to the type of the products they enter.
template <typename T, int kAct>
__global__ void __launch_bounds__(kThreads) k_slopes(const Slopes a, long long blocks, unsigned row_blocks) {
  for (long long block = blockIdx.x; block < blocks; block += gridDim.x) {
    const long long row = block / row_blocks;
    const int at = (int)((unsigned)(block - row * row_blocks) * kThreads + threadIdx.x) * kSlopeVec;
    if (at >= a.hidden) continue;
    const T *grad = static_cast<const T *>(a.grad_out) + row * a.grad_out_stride + at;
    const long long kept = row * a.kept_stride + at;
    float gate_scale = 0, up_scale = 0;
    if (a.gate_scales != nullptr) {
      const long long group = row * ((a.hidden + kScaleGroup - 1) / kScaleGroup) + at / kScaleGroup;
      gate_scale = a.gate_scales[group];
      up_scale = a.up_scales[group];
    }
    T dg[kSlopeVec], du[kSlopeVec];
#pragma unroll
    for (int c = 0; c < kSlopeVec; ++c) {
      const bool held = at + c < a.hidden;
      const float y = held ? (float)grad[c] : 0.0f;
      float g, u;
      if (a.gate_scales != nullptr) {
        g = held ? Restored(static_cast<const signed char *>(a.gate)[kept + c], gate_scale) : 0.0f;
        u = held ? Restored(static_cast<const signed char *>(a.up)[kept + c], up_scale) : 0.0f;
      } else {
        g = held ? (float)static_cast<const T *>(a.gate)[kept + c] : 0.0f;
        u = held ? (float)static_cast<const T *>(a.up)[kept + c] : 0.0f;
      }
      float act, slope;
      ActAndSlope<kAct>(g, &act, &slope);
      dg[c] = Round<T>(y * u * slope);
      du[c] = Round<T>(y * act);
    }
    StoreFour<T>(static_cast<T *>(a.d_gate) + row * a.d_stride, at, a.hidden, dg);
    StoreFour<T>(static_cast<T *>(a.d_up) + row * a.d_stride, at, a.hidden, du);
  }
}

// ------------------------------------------------------------------ the host

constexpr long long kMostGrid = 1 << 20;

long long Pieces(long long n, long long of) { return (n + of - 1) / of; }

struct Plan {
  long long d_stride, x_splits, x_split_blocks, w_splits, w_split_blocks;
  size_t d_bytes, bytes;
};

// Few tiles share out their k's until the chip is full; a share is at least eight blocks.
void SetSplits(long long tiles, long long blocks, long long *splits, long long *split_blocks) {
  const long long most = std::max<long long>(1, std::min({512 / std::max<long long>(tiles, 1), blocks / 8, 64ll}));
  *split_blocks = std::max<long long>(1, Pieces(blocks, most));
  *splits = std::max<long long>(1, Pieces(blocks, *split_blocks));
}

void CheckLayerSizes(long long rows, int dim, int hidden, int type) {
  CheckType(type);
  if (rows < 0 || rows >= (1ll << 31)) throw std::runtime_error("bad number of rows");
  if (dim < 1 || dim > (1 << 24)) throw std::runtime_error("bad dimension");
  if (hidden < 1 || hidden > (1 << 24)) throw std::runtime_error("bad hidden dimension");
}

Plan PlanOf(long long rows, int dim, int hidden, int type) {
  const long long item = (long long)ElementBytes(type), k = kTileBytes / item;
  Plan p;
  p.d_stride = Pieces(hidden, 64) * 64;
  SetSplits(Pieces(rows, kTile) * Pieces(dim, kTile), 2 * Pieces(hidden, k), &p.x_splits, &p.x_split_blocks);
  SetSplits(2 * Pieces(hidden, kTile) * Pieces(dim, kTile), Pieces(rows, k), &p.w_splits, &p.w_split_blocks);
  p.d_bytes = (size_t)(rows * p.d_stride * item + 255) / 256 * 256;
  const size_t partial = std::max<size_t>(p.x_splits > 1 ? (size_t)p.x_splits * rows * dim * 4 : 0, p.w_splits > 1 ? (size_t)p.w_splits * 2 * hidden * dim * 4 : 0);
  p.bytes = 2 * p.d_bytes + partial;
  return p;
}

void CheckStride(long long stride, long long width, long long rows, const char *what) {
  if (stride < 0 || stride >= (1ll << 31) || (rows > 1 && stride < width)) throw std::runtime_error(std::string("bad stride of ") + what);
}

// (checks what both directions take; kept: whether gate and up must be there)
void CheckLayer(const GatedLayer &l, bool kept, size_t need) {
  CheckLayerSizes(l.rows, l.dim, l.hidden, l.type);
  if (l.activation != kSilu && l.activation != kGelu) throw std::runtime_error("unknown activation");
  CheckStride(l.x_stride, 0, l.rows, "x");
  CheckStride(l.w_stride, 0, l.hidden, "the weights");
  if (!l.w_gate || !l.w_up || (l.rows > 0 && !l.x)) throw std::runtime_error("null pointer argument");
  if ((l.gate == nullptr) != (l.up == nullptr) || (l.gate_scales == nullptr) != (l.up_scales == nullptr)) throw std::runtime_error("gate and up go together");
  if (l.gate_scales && !l.gate) throw std::runtime_error("scales without gate and up");
  if (kept && l.rows > 0 && !l.gate) throw std::runtime_error("null pointer argument");
  if (l.gate) CheckStride(l.kept_stride, l.hidden, l.rows, "gate and up");
  const size_t item = ElementBytes(l.type);
  CheckAligned(l.x, item, "x");
  CheckAligned(l.w_gate, item, "w_gate");
  CheckAligned(l.w_up, item, "w_up");
  if (!l.gate_scales) CheckAligned(l.gate, item, "gate"), CheckAligned(l.up, item, "up");
  CheckAligned(l.gate_scales, 4, "gate_scales");
  CheckAligned(l.up_scales, 4, "up_scales");
  if (need > 0) {
    if (!l.work) throw std::runtime_error("null pointer argument");
    CheckAligned(l.work, 16, "work");
    if (l.work_bytes < need) throw std::runtime_error("work memory is too small: " + std::to_string(need) + " bytes are needed");
  }
}

template <typename Fn>
void WithActivation(int activation, Fn &&fn) {
  if (activation == kSilu) fn(std::integral_constant<int, kSilu>());
  else fn(std::integral_constant<int, kGelu>());
}

template <typename T, bool kAcrossA, bool kAcrossB>
void Launch(const Products &p, hipStream_t stream) {
  const int columns = (int)Pieces(p.columns, kTile);
  const long long each = Pieces(p.rows, kTile) * columns, tiles = each * p.batch * p.splits;
  hipLaunchKernelGGL((k_products<T, kAcrossA, kAcrossB>), dim3((unsigned)std::min(tiles, kMostGrid)), dim3(kThreads), 0, stream, p, tiles, columns, each);
  if (p.splits > 1) {
    const long long blocks = Pieces(p.rows * p.columns * p.batch, kThreads);
    hipLaunchKernelGGL((k_products_join<T>), dim3((unsigned)std::min(blocks, kMostGrid)), dim3(kThreads), 0, stream, p);
  }
}

}  // namespace

size_t GatedBytes(long long rows, int dim, int hidden, int type) {
  CheckLayerSizes(rows, dim, hidden, type);
  return 0;
}

void Gated(const GatedArgs &a) {
  const GatedLayer &l = a.layer;
  CheckLayer(l, false, GatedBytes(l.rows, l.dim, l.hidden, l.type));
  CheckStride(a.out_stride, l.hidden, l.rows, "out");
  CheckAligned(a.out, ElementBytes(l.type), "out");
  if (l.rows == 0) return;
  if (!a.out) throw std::runtime_error("null pointer argument");
  OnDeviceOf device(a.out);
  const Forward f{l.x, l.w_gate, l.w_up, l.rows, l.dim, l.hidden, l.x_stride, l.w_stride, a.out, a.out_stride, l.gate, l.up, l.gate_scales,
                  l.up_scales, l.kept_stride};
  const int columns = (int)Pieces(l.hidden, kHalf);
  const long long tiles = Pieces(l.rows, kTile) * columns;
  WithType(l.type, [&](auto type) {
    WithActivation(l.activation, [&](auto act) {
      hipLaunchKernelGGL((k_gated<decltype(type), decltype(act)::value>), dim3((unsigned)std::min(tiles, kMostGrid)), dim3(kThreads), 0,
                         static_cast<hipStream_t>(l.stream), f, tiles, columns);
    });
  });
  HIP_OK(hipGetLastError());
}

size_t GatedGradBytes(long long rows, int dim, int hidden, int type) {
  CheckLayerSizes(rows, dim, hidden, type);
  return PlanOf(rows, dim, hidden, type).bytes;
}

void GatedGrad(const GatedGradArgs &a) {
  const GatedLayer &l = a.layer;
  const Plan plan = (CheckLayerSizes(l.rows, l.dim, l.hidden, l.type), PlanOf(l.rows, l.dim, l.hidden, l.type));
  CheckLayer(l, true, plan.bytes);
  if ((a.grad_w_gate == nullptr) != (a.grad_w_up == nullptr)) throw std::runtime_error("the gradients of both weights go together");
  const size_t item = ElementBytes(l.type);
  CheckAligned(a.grad_out, item, "grad_out");
  CheckAligned(a.grad_x, item, "grad_x");
  CheckAligned(a.grad_w_gate, item, "grad_w_gate");
  CheckAligned(a.grad_w_up, item, "grad_w_up");
  CheckStride(a.grad_out_stride, 0, l.rows, "grad_out");
  if (a.grad_x) CheckStride(a.grad_x_stride, l.dim, l.rows, "grad_x");
  if (a.grad_w_gate) CheckStride(a.grad_w_stride, l.dim, l.hidden, "the weights' gradients");
  if (l.rows > 0 && !a.grad_out) throw std::runtime_error("null pointer argument");
  if (!a.grad_w_gate && (!a.grad_x || l.rows == 0)) return;
  OnDeviceOf device(a.grad_w_gate ? a.grad_w_gate : a.grad_x);
  const hipStream_t stream = static_cast<hipStream_t>(l.stream);
  unsigned char *work = static_cast<unsigned char *>(l.work);
  void *d_gate = work, *d_up = work + plan.d_bytes;
  float *partial = reinterpret_cast<float *>(work + 2 * plan.d_bytes);
  WithType(l.type, [&](auto type) {
    typedef decltype(type) T;
    if (l.rows > 0) {
      const Slopes s{a.grad_out, a.grad_out_stride, l.gate, l.up, l.gate_scales, l.up_scales, l.kept_stride, d_gate, d_up, plan.d_stride, l.rows, l.hidden};
      const unsigned row_blocks = (unsigned)Pieces(l.hidden, kThreads * kSlopeVec);
      const long long blocks = l.rows * row_blocks;
      WithActivation(l.activation, [&](auto act) {
        hipLaunchKernelGGL((k_slopes<T, decltype(act)::value>), dim3((unsigned)std::min(blocks, kMostGrid)), dim3(kThreads), 0, stream, s, blocks, row_blocks);
      });
    }
    if (a.grad_x && l.rows > 0)
      Launch<T, false, true>(Products{{{d_gate, d_up}, plan.d_stride}, {{l.w_gate, l.w_up}, l.w_stride}, l.rows, l.dim, l.hidden, 2, 1, {a.grad_x, nullptr},
                                      a.grad_x_stride, (int)plan.x_splits, plan.x_split_blocks, partial}, stream);
    if (a.grad_w_gate)
      Launch<T, true, true>(Products{{{d_gate, d_up}, plan.d_stride}, {{l.x, l.x}, l.x_stride}, l.hidden, l.dim, l.rows, 1, 2,
                                     {a.grad_w_gate, a.grad_w_up}, a.grad_w_stride, (int)plan.w_splits, plan.w_split_blocks, partial}, stream);
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
