// Embedding lookup over bags of tokens and the gradient of its table by sorted tokens.
//
//   lookup    out[i]        = scale * sum_j table[token(i, j)]
//   gradient  grad_table[v] = scale * sum of grad_out[i] over all (i, j) with token(i, j) = v
//
// The gradient gathers: the (token, bag) pairs are put in order of tokens first (a stable radix sort), so that every sum is
// formed in an order that depends on the tokens alone, and no atomic decides it.
#include <algorithm>
#include <cstring>
#include <limits>

#include "operators_device.h"

namespace arb {
namespace {

// ------------------------------------------------------------------ lookup

template <typename Token>
struct Bags {
  const Token *tokens;
  long long n;
  long long token_stride, bag_stride;
  int bag;
  unsigned vocab;
  unsigned *status;
  // The row of the table that token j of bag i names; `vocab` for none.
  __device__ __forceinline__ unsigned At(long long i, long long j) const {
    const long long t = tokens[i * token_stride + j * bag_stride];
    if (t >= 0 && t < (long long)vocab) return (unsigned)t;
    if (t != -1 && status != nullptr) *status = 1u;
    return vocab;
  }
};

template <typename Token>
Bags<Token> BagsOf(const TokenBags &b) {
  return Bags<Token>{static_cast<const Token *>(b.tokens), b.n, b.token_stride, b.bag_stride, b.bag, (unsigned)b.vocab, b.status};
}

constexpr int kThreads = 256;

template <typename T, typename Token>
__global__ void __launch_bounds__(kThreads)
k_embedding(const Bags<Token> bags, const T *__restrict__ table, long long table_stride, T *__restrict__ out, long long out_stride,
            int dim, float scale) {
  const long long all = bags.n * dim;
  for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < all; e += (long long)gridDim.x * kThreads) {
    const long long i = e / dim;
    const int d = (int)(e - i * dim);
    float sum = 0.0f;
    for (int j = 0; j < bags.bag; ++j) {
      const unsigned t = bags.At(i, j);
      if (t < bags.vocab) sum += static_cast<float>(table[(long long)t * table_stride + d]);
    }
    out[i * out_stride + d] = Round<T>(sum * scale);
  }
}

// -------------------------------------------------------------------- sort
//
// Least significant digit first, up to 9 bits at a time: two passes up to a vocabulary of 262,143.  A tile of 4096 pairs is put in
// order in the LDS, so that the pairs of a digit leave as one run.

constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kSortRounds = 8;                         // pairs per thread
constexpr int kSortTile = kSortThreads * kSortRounds;  // 4096
constexpr int kWavePairs = kSortTile / kSortWaves;
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;

// Where a pass takes its pairs from: the tokens themselves, or keys and rows.
template <typename Token>
struct FromTokens {
  Bags<Token> bags;
  unsigned m;
  bool by_column;  // pair p is token p / n of bag p % n, else token p % bag of bag p / bag
  __device__ __forceinline__ void Get(unsigned p, unsigned *key, unsigned *row) const {
    unsigned i, j;
    if (by_column) {
      j = p / (unsigned)bags.n;
      i = p - j * (unsigned)bags.n;
    } else {
      i = p / (unsigned)bags.bag;
      j = p - i * (unsigned)bags.bag;
    }
    *key = bags.At(i, j);
    *row = i;
  }
};
struct FromPairs {
  const unsigned *keys, *rows;
  unsigned m;
  __device__ __forceinline__ void Get(unsigned p, unsigned *key, unsigned *row) const {
    *key = keys[p];
    *row = rows[p];
  }
};

struct Digit {
  int shift;
  unsigned mask;
  __device__ __forceinline__ unsigned Of(unsigned key) const { return (key >> shift) & mask; }
};

// Digit counts of one tile: counts[digit * tiles + tile].
template <typename Source>
__global__ void __launch_bounds__(kSortThreads) k_sort_count(const Source in, const Digit digit, unsigned *__restrict__ counts, unsigned tiles) {
  __shared__ unsigned s_count[kDigits];
  s_count[threadIdx.x] = 0;
  __syncthreads();
  const unsigned base = blockIdx.x * kSortTile;
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const unsigned p = base + k * kSortThreads + threadIdx.x;
    if (p < in.m) {
      unsigned key, row;
      in.Get(p, &key, &row);
      atomicAdd(&s_count[digit.Of(key)], 1u);
    }
  }
  __syncthreads();
  counts[(size_t)threadIdx.x * tiles + blockIdx.x] = s_count[threadIdx.x];
}

// Exclusive scan of the tile counts of a digit, in place, and the digit's total.  A workgroup per digit.
__global__ void __launch_bounds__(256) k_sort_scan(unsigned *__restrict__ counts, unsigned tiles, unsigned *__restrict__ totals) {
  __shared__ unsigned s_wave[4];
  unsigned *v = counts + (size_t)blockIdx.x * tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned carry = 0;
  for (unsigned base = 0; base < tiles; base += 256) {
    const unsigned i = base + threadIdx.x;
    const unsigned c = i < tiles ? v[i] : 0u;
    unsigned incl = c;
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned o = __shfl_up(incl, off);
      if (lane >= off) incl += o;
    }
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    unsigned before = carry;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += s_wave[w];
      carry += s_wave[w];
    }
    if (i < tiles) v[i] = before + incl - c;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Lanes of the wave that hold the same digit as this one.
__device__ __forceinline__ unsigned long long DigitPeers(unsigned d, bool valid) {
  unsigned long long peers = __ballot(valid);
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const unsigned long long m = __ballot((d >> b) & 1u);
    peers &= ((d >> b) & 1u) ? m : ~m;
  }
  return peers;
}

// Stable scatter of one tile.  counts (scanned): pairs of the same digit in the tiles before.
template <typename Source>
__global__ void __launch_bounds__(kSortThreads)
k_sort_scatter(const Source in, const Digit digit, const unsigned *__restrict__ counts, unsigned tiles, const unsigned *__restrict__ totals,
               unsigned *__restrict__ keys, unsigned *__restrict__ rows) {
  __shared__ unsigned s_key[kSortTile], s_row[kSortTile];
  __shared__ unsigned s_wave[kSortWaves][kDigits];  // pairs of each digit of a wave; then those of the waves before
  __shared__ unsigned s_first[kDigits];             // place in the tile of the first pair of each digit
  __shared__ unsigned s_out[kDigits];               // output position of that pair
  __shared__ unsigned s_sum[2][kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned base = blockIdx.x * kSortTile, held = min((unsigned)kSortTile, in.m - base);
  for (int w = 0; w < kSortWaves; ++w) s_wave[w][threadIdx.x] = 0;
  unsigned key[kSortRounds], row[kSortRounds], rank[kSortRounds];
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const unsigned i = wave * kWavePairs + k * 64 + lane;
    key[k] = row[k] = 0;
    if (i < held) in.Get(base + i, &key[k], &row[k]);
  }
  const unsigned total = totals[threadIdx.x], before = counts[(size_t)threadIdx.x * tiles + blockIdx.x];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const bool valid = wave * kWavePairs + k * 64 + lane < held;
    const unsigned d = digit.Of(key[k]);
    const unsigned long long peers = DigitPeers(d, valid);
    const unsigned below = (unsigned)__popcll(peers & ((1ull << lane) - 1ull));
    const unsigned held_of = s_wave[wave][d];
    rank[k] = held_of + below;
    __builtin_amdgcn_wave_barrier();  // every lane has read its counter
    if (valid && below == 0) s_wave[wave][d] = held_of + (unsigned)__popcll(peers);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  {
    // thread = digit: pairs of smaller digits in the tile, and in all
    unsigned mine = 0;
    for (int w = 0; w < kSortWaves; ++w) {
      const unsigned c = s_wave[w][threadIdx.x];
      s_wave[w][threadIdx.x] = mine;
      mine += c;
    }
    unsigned in_tile = mine, in_all = total;
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned a = __shfl_up(in_tile, off), b = __shfl_up(in_all, off);
      if (lane >= off) {
        in_tile += a;
        in_all += b;
      }
    }
    if (lane == 63) {
      s_sum[0][wave] = in_tile;
      s_sum[1][wave] = in_all;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      in_tile += s_sum[0][w];
      in_all += s_sum[1][w];
    }
    s_first[threadIdx.x] = in_tile - mine;
    s_out[threadIdx.x] = in_all - total + before;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    if (wave * kWavePairs + k * 64 + lane < held) {
      const unsigned d = digit.Of(key[k]);
      const unsigned at = s_first[d] + s_wave[wave][d] + rank[k];
      s_key[at] = key[k];
      s_row[at] = row[k];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const unsigned i = k * kSortThreads + threadIdx.x;
    if (i < held) {
      const unsigned d = digit.Of(s_key[i]);
      const unsigned to = s_out[d] + (i - s_first[d]);
      keys[to] = s_key[i];
      rows[to] = s_row[i];
    }
  }
}

// Passes and bits of a digit for keys in [0, vocab].
struct SortPlan {
  int passes, bits;
  unsigned m, tiles;
  size_t counts_bytes, pairs_bytes, bytes;
};
constexpr size_t Align256(size_t v) { return (v + 255) / 256 * 256; }

SortPlan PlanSort(long long n, int bag, long long vocab) {
  SortPlan s;
  int bits = 1;
  while (vocab >> bits) ++bits;
  s.passes = (bits + kDigitBits - 1) / kDigitBits;
  s.bits = (bits + s.passes - 1) / s.passes;
  s.m = (unsigned)(n * bag);
  s.tiles = (s.m + kSortTile - 1) / kSortTile;
  s.counts_bytes = Align256((size_t)s.tiles * kDigits * sizeof(unsigned));
  s.pairs_bytes = s.passes > 1 ? Align256((size_t)s.m * sizeof(unsigned)) : 0;
  s.bytes = s.counts_bytes + kDigits * sizeof(unsigned) + 2 * s.pairs_bytes;
  return s;
}

// ---------------------------------------------------------------- gradient

// First pair whose key is at least v.
__device__ __forceinline__ unsigned LowerBound(const unsigned *__restrict__ keys, unsigned m, unsigned v) {
  unsigned low = 0, high = m;
  while (low < high) {
    const unsigned mid = (low + high) / 2;
    if (keys[mid] < v) low = mid + 1;
    else high = mid;
  }
  return low;
}

template <typename T, typename O>
__global__ void __launch_bounds__(kThreads)
k_embedding_grad(const unsigned *__restrict__ keys, const unsigned *__restrict__ rows, unsigned m, unsigned n, long long vocab,
                 const T *__restrict__ grad_out, long long out_stride, O *__restrict__ grad_table, long long table_stride, int dim,
                 float scale, bool accumulate) {
  for (long long v = blockIdx.x; v < vocab; v += gridDim.x) {
    const unsigned begin = LowerBound(keys, m, (unsigned)v), end = LowerBound(keys, m, (unsigned)v + 1u);
    if (accumulate && begin == end) continue;
    for (int d = threadIdx.x; d < dim; d += kThreads) {
      float sum = 0.0f;
      for (unsigned p = begin; p < end; ++p)
        if (rows[p] < n) sum += static_cast<float>(grad_out[(long long)rows[p] * out_stride + d]);
      sum = begin < end ? sum * scale : 0.0f;
      O *at = grad_table + v * table_stride + d;
      *at = Round<O>(accumulate ? static_cast<float>(*at) + sum : sum);
    }
  }
}

// ------------------------------------------------------------------ checks

void CheckShape(long long n, int bag, long long vocab) {
  if (n < 0 || bag < 0) throw std::runtime_error("bad row count or bag size");
  if (n >= (1ll << 31) || (bag > 0 && n > ((1ll << 31) - 1) / bag)) throw std::runtime_error("too many tokens: n * bag must be below 2^31");
  if (vocab < 1 || vocab >= (1ll << 31)) throw std::runtime_error("bad vocabulary size");
}

void CheckTokens(const TokenBags &b) {
  CheckShape(b.n, b.bag, b.vocab);
  if (b.bits != 32 && b.bits != 64) throw std::runtime_error("tokens have 32 or 64 bits");
  if (b.token_stride < 0 || b.bag_stride < 0) throw std::runtime_error("bad token stride");
  if (b.n * b.bag > 0 && !b.tokens) throw std::runtime_error("null pointer argument");
  CheckAligned(b.tokens, b.bits / 8, "tokens");
  CheckAligned(b.status, 4, "status");
}

// Rows [0, n) of `dim` elements, `stride` apart.
void CheckRows(const void *p, long long n, long long stride, int dim, int type, bool apart, const char *what) {
  if (dim < 1) throw std::runtime_error("bad dimension");
  if (stride < 0 || (apart && n > 1 && stride < dim)) throw std::runtime_error(std::string("rows of ") + what + " overlap");
  if (n > 0 && !p) throw std::runtime_error("null pointer argument");
  CheckAligned(p, ElementBytes(type), what);
}

template <typename Fn>
void WithToken(int bits, Fn &&fn) {
  if (bits == 32) fn(int());
  else fn((long long)0);
}

}  // namespace

void Embedding(const EmbeddingArgs &a) {
  CheckType(a.type);
  CheckTokens(a.bags);
  CheckRows(a.table, a.bags.vocab, a.table_stride, a.dim, a.type, false, "table");
  CheckRows(a.out, a.bags.n, a.out_stride, a.dim, a.type, true, "out");
  if (a.bags.n == 0) return;
  OnDeviceOf device(a.out);
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const unsigned grid = (unsigned)std::min<long long>((a.bags.n * a.dim + kThreads - 1) / kThreads, 1 << 16);
  WithType(a.type, [&](auto e) {
    WithToken(a.bags.bits, [&](auto token) {
      typedef decltype(e) T;
      typedef decltype(token) Token;
      hipLaunchKernelGGL((k_embedding<T, Token>), dim3(grid), dim3(kThreads), 0, st, BagsOf<Token>(a.bags), static_cast<const T *>(a.table),
                         a.table_stride, static_cast<T *>(a.out), a.out_stride, a.dim, a.scale);
    });
  });
  HIP_OK(hipGetLastError());
}

size_t EmbeddingSortBytes(long long n, int bag, long long vocab) {
  CheckShape(n, bag, vocab);
  return PlanSort(n, bag, vocab).bytes;
}

void EmbeddingSort(const EmbeddingSortArgs &a) {
  CheckTokens(a.bags);
  const SortPlan plan = PlanSort(a.bags.n, a.bags.bag, a.bags.vocab);
  if (plan.m == 0) return;
  if (!a.keys || !a.rows || !a.work) throw std::runtime_error("null pointer argument");
  CheckAligned(a.keys, 4, "keys");
  CheckAligned(a.rows, 4, "rows");
  CheckAligned(a.work, 16, "work memory");
  if (a.work_bytes < plan.bytes) throw std::runtime_error("work memory too small");
  OnDeviceOf device(a.keys);
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  unsigned char *work = static_cast<unsigned char *>(a.work);
  unsigned *counts = reinterpret_cast<unsigned *>(work);
  unsigned *totals = reinterpret_cast<unsigned *>(work + plan.counts_bytes);
  unsigned *spare[2];
  spare[0] = totals + kDigits;
  spare[1] = spare[0] + plan.pairs_bytes / sizeof(unsigned);
  unsigned *last[2] = {a.keys, a.rows};
  for (int pass = 0; pass < plan.passes; ++pass) {
    // the last pass writes to the caller's arrays, the passes before it in turn
    unsigned **to = (plan.passes - 1 - pass) % 2 == 0 ? last : spare, **from = to == last ? spare : last;
    const Digit digit{pass * plan.bits, (1u << plan.bits) - 1u};
    auto launch = [&](const auto &in) {
      typedef std::decay_t<decltype(in)> Source;
      hipLaunchKernelGGL((k_sort_count<Source>), dim3(plan.tiles), dim3(kSortThreads), 0, st, in, digit, counts, plan.tiles);
      hipLaunchKernelGGL(k_sort_scan, dim3(kDigits), dim3(256), 0, st, counts, plan.tiles, totals);
      hipLaunchKernelGGL((k_sort_scatter<Source>), dim3(plan.tiles), dim3(kSortThreads), 0, st, in, digit, counts, plan.tiles, totals, to[0],
                         to[1]);
    };
    if (pass > 0) {
      launch(FromPairs{from[0], from[1], plan.m});
    } else {
      // pairs in the order the tokens lie in memory
      const bool by_column = a.bags.token_stride < a.bags.bag_stride;
      WithToken(a.bags.bits, [&](auto token) {
        typedef decltype(token) Token;
        launch(FromTokens<Token>{BagsOf<Token>(a.bags), plan.m, by_column});
      });
    }
  }
  HIP_OK(hipGetLastError());
}

size_t EmbeddingGradBytes(long long n, int bag, int dim) {
  CheckShape(n, bag, 1);
  if (dim < 1) throw std::runtime_error("bad dimension");
  return 256;
}

void EmbeddingGrad(const EmbeddingGradArgs &a) {
  CheckType(a.type);
  CheckType(a.table_type);
  if (a.table_type != kFloat32 && a.table_type != a.type) throw std::runtime_error("the table's gradient is float32 or of the type of grad_out");
  CheckShape(a.n, a.bag, a.vocab);
  CheckRows(a.grad_out, a.n, a.out_stride, a.dim, a.type, false, "grad_out");
  CheckRows(a.grad_table, a.vocab, a.table_stride, a.dim, a.table_type, true, "grad_table");
  const unsigned m = (unsigned)(a.n * a.bag);
  if (m > 0 && (!a.keys || !a.rows || !a.work)) throw std::runtime_error("null pointer argument");
  CheckAligned(a.keys, 4, "keys");
  CheckAligned(a.rows, 4, "rows");
  CheckAligned(a.work, 16, "work memory");
  if (m > 0 && a.work_bytes < EmbeddingGradBytes(a.n, a.bag, a.dim)) throw std::runtime_error("work memory too small");
  OnDeviceOf device(a.grad_table);
  hipStream_t st = static_cast<hipStream_t>(a.stream);
  const unsigned grid = (unsigned)std::min<long long>(a.vocab, 1 << 16);
  auto launch = [&](auto t, auto o) {
    typedef decltype(t) T;
    typedef decltype(o) O;
    hipLaunchKernelGGL((k_embedding_grad<T, O>), dim3(grid), dim3(kThreads), 0, st, a.keys, a.rows, m, (unsigned)a.n, a.vocab, static_cast<const T *>(a.grad_out),
                       a.out_stride, static_cast<O *>(a.grad_table), a.table_stride, a.dim, a.scale, a.accumulate);
  };
  WithType(a.type, [&](auto t) {
    if (a.table_type == kFloat32) launch(t, float());
    else launch(t, t);
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
