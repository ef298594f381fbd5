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
#include <type_traits>

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
    return Row(tokens[i * token_stride + j * bag_stride]);
  }
  __device__ __forceinline__ unsigned Row(Token t) const {
    typedef std::make_unsigned_t<Token> Word;
    if ((Word)t < (Word)vocab) return (unsigned)t;
    if (t != -1 && status != nullptr) *status = 1u;
    return vocab;
  }
};

template <typename Token>
Bags<Token> BagsOf(const TokenBags &b) {
  return Bags<Token>{static_cast<const Token *>(b.tokens), b.n, b.token_stride, b.bag_stride, b.bag, (unsigned)b.vocab, b.status};
}

constexpr int kThreads = 256;
constexpr int kNarrow = 8;           // widest row that a lane holds whole in the gradient
constexpr unsigned kMostSlots = 256;  // table rows whose zeros a workgroup writes

// kVec elements of a row from `at` on, of which `held` are in it; what is not held is 0 (Load) and left alone (Store).
template <typename T, int kVec>
__device__ __forceinline__ void Load(const T *__restrict__ at, int held, Pack<T, kVec> *to) {
  if (held >= kVec) {
    *to = *reinterpret_cast<const Pack<T, kVec> *>(at);
  } else {
#pragma unroll
    for (int c = 0; c < kVec; ++c) to->v[c] = c < held ? at[c] : T(0);
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void Store(T *__restrict__ at, int held, const Pack<T, kVec> &from) {
  if (held >= kVec) {
    *reinterpret_cast<Pack<T, kVec> *>(at) = from;
  } else {
#pragma unroll
    for (int c = 0; c < kVec; ++c)
      if (c < held) at[c] = from.v[c];
  }
}

// Rows of the two matrices of a lookup.
template <typename T>
struct Rows {
  const T *table;
  long long table_stride;
  T *out;
  long long out_stride;
  int dim;
  float scale;
};

// Bags of one token: rows are copied, scaled.  2^lanes_log lanes take a piece of kPieces vectors a lane of a row, so that all
// its loads are in flight at once (blockIdx.y: which piece).
constexpr int kPieces = 4;
template <typename T, int kVec, typename Token>
__global__ void __launch_bounds__(kThreads) k_embedding_one(const Bags<Token> bags, const Rows<T> r, int lanes_log) {
  const long long i = (long long)(((unsigned long long)blockIdx.x * kThreads + threadIdx.x) >> lanes_log);
  if (i >= bags.n) return;
  const unsigned lane = threadIdx.x & ((1u << lanes_log) - 1u);
  const int step = kVec << lanes_log;
  const int first = (int)blockIdx.y * (step * kPieces) + (int)lane * kVec;
  const unsigned t = bags.At(i, 0);
  const T *from = r.table + (long long)t * r.table_stride;
  T *to = r.out + i * r.out_stride;
  Pack<T, kVec> x[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int d = first + k * step;
    if (t < bags.vocab) Load<T, kVec>(from + d, r.dim - d, &x[k]);
    else
#pragma unroll
      for (int c = 0; c < kVec; ++c) x[k].v[c] = T(0);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int d = first + k * step;
#pragma unroll
    for (int c = 0; c < kVec; ++c) x[k].v[c] = Round<T>(static_cast<float>(x[k].v[c]) * r.scale);
    if (d < r.dim) Store<T, kVec>(to + d, r.dim - d, x[k]);
  }
}

// Bags of several tokens.  A row of the result is 2^lanes_log lanes wide (kVec elements a lane), and 2^shares_log shares of
// them take every so many-th token each and meet in the end, by steps of halves.  kAhead tokens of a lane are in flight.
constexpr int kAhead = 8;
template <typename T, int kVec, typename Token>
__global__ void __launch_bounds__(kThreads)
k_embedding_bag(const Bags<Token> bags, const Rows<T> r, int lanes_log, int shares_log) {
  const long long i = (long long)(((unsigned long long)blockIdx.x * kThreads + threadIdx.x) >> (lanes_log + shares_log));
  const bool live = i < bags.n;
  const unsigned lane = threadIdx.x & ((1u << lanes_log) - 1u);
  const int share = (int)((threadIdx.x >> lanes_log) & ((1u << shares_log) - 1u)), shares = 1 << shares_log;
  const int d = ((int)blockIdx.y << lanes_log) * kVec + (int)lane * kVec;
  float sum[kVec];
#pragma unroll
  for (int c = 0; c < kVec; ++c) sum[c] = 0.0f;
  if (live && d < r.dim) {
    const Token *at = bags.tokens + i * bags.token_stride + share * bags.bag_stride;
    const long long step = (long long)shares * bags.bag_stride;
    for (int j = share; j < bags.bag; j += kAhead * shares) {
      unsigned t[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        t[k] = bags.vocab;
        if (j + k * shares < bags.bag) t[k] = bags.Row(at[k * step]);
      }
      at += kAhead * step;
      Pack<T, kVec> x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
#pragma unroll
        for (int c = 0; c < kVec; ++c) x[k].v[c] = T(0);
        if (t[k] < bags.vocab) Load<T, kVec>(r.table + (long long)t[k] * r.table_stride + d, r.dim - d, &x[k]);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int c = 0; c < kVec; ++c) sum[c] += static_cast<float>(x[k].v[c]);
    }
  }
  for (int s = shares_log - 1; s >= 0; --s)
#pragma unroll
    for (int c = 0; c < kVec; ++c) sum[c] += __shfl_xor(sum[c], 1 << (lanes_log + s));
  if (live && share == 0 && d < r.dim) {
    Pack<T, kVec> y;
#pragma unroll
    for (int c = 0; c < kVec; ++c) y.v[c] = Round<T>(sum[c] * r.scale);
    Store<T, kVec>(r.out + i * r.out_stride + d, r.dim - d, y);
  }
}

int LogAtLeast(long long v) {
  int log = 0;
  while ((1ll << log) < v) ++log;
  return log;
}

template <typename T, int kVec, typename Token>
void LaunchLookup(const EmbeddingArgs &a, hipStream_t st) {
  const Bags<Token> bags = BagsOf<Token>(a.bags);
  const Rows<T> r{static_cast<const T *>(a.table), a.table_stride, static_cast<T *>(a.out), a.out_stride, a.dim, a.scale};
  const long long vectors = (a.dim + kVec - 1) / kVec;
  const int lanes_log = std::min(LogAtLeast(vectors), 6);
  long long per_row = (vectors + (1ll << lanes_log) - 1) >> lanes_log;  // pieces of a row
  int group_log = lanes_log, shares_log = 0;
  if (a.bags.bag == 1) {
    per_row = (per_row + kPieces - 1) / kPieces;
  } else {
    // Where the tokens of a bag lie beside each other the lanes of a wave read along them; otherwise they read along the
    // bags, unless these do not fill the chip (4 waves a CU).
    const int most = std::min(6 - lanes_log, LogAtLeast((a.bags.bag + 15) / 16));
    if (a.bags.bag_stride <= a.bags.token_stride) shares_log = most;
    else
      while (shares_log < most && ((a.bags.n * per_row) << (lanes_log + shares_log)) < 65536) ++shares_log;
    group_log += shares_log;
  }
  const long long blocks = ((a.bags.n << group_log) + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)blocks, (unsigned)per_row);
  if (a.bags.bag == 1) hipLaunchKernelGGL((k_embedding_one<T, kVec, Token>), grid, dim3(kThreads), 0, st, bags, r, lanes_log);
  else hipLaunchKernelGGL((k_embedding_bag<T, kVec, Token>), grid, dim3(kThreads), 0, st, bags, r, lanes_log, shares_log);
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
//
// The sorted pairs are cut into chunks of equal length, whatever the tokens are: a token that half of all bags name is
// the work of many waves.  A run of equal keys inside one chunk is summed and written there; of a run that goes on beyond its
// chunk each chunk leaves its part of the sum in the work memory, and a second launch (k_grad_join) adds the parts in order.

// First pair whose key is at least v: the whole wave asks, 64 probes a step (five steps for 2^30 pairs, where halving takes thirty loads
// one after the other).
__device__ __forceinline__ unsigned WaveLowerBound(const unsigned *__restrict__ keys, unsigned m, unsigned v) {
  unsigned low = 0, high = m;  // the answer is in [low, high]
  while (low < high) {
    const unsigned step = (high - low + 63u) / 64u, at = low + (threadIdx.x & 63u) * step;
    const unsigned long long less = __ballot(at < high && keys[at] < v);
    if (less == 0ull) return low;
    const unsigned last = 63u - (unsigned)__clzll((long long)less);  // probes are in order, so `less` is a run from lane 0
    const unsigned next = low + (last + 1u) * step;
    low = low + last * step + 1u;
    high = min(high, next);
  }
  return low;
}

template <typename T, typename O>
struct Gradient {
  const unsigned *keys, *rows;
  unsigned m, n, vocab;
  const T *grad_out;
  long long out_stride;
  O *grad_table;
  long long table_stride;
  int dim;
  float scale;
  bool accumulate;
  unsigned chunk, chunks;  // pairs of a chunk; chunks
  float *parts;            // [chunks][2][dim]: the sum of the run that comes in, of the one that goes on
  unsigned fill_blocks, slots;  // workgroups that write the rows no token names, rows of each
  int lanes_log;
  unsigned pieces;

  template <int kVec>
  __device__ __forceinline__ void Write(unsigned v, int d, const float (&sum)[kVec]) const {
    O *at = grad_table + (long long)v * table_stride + d;
    Pack<O, kVec> y;
    if (accumulate) Load<O, kVec>(at, dim - d, &y);
#pragma unroll
    for (int c = 0; c < kVec; ++c) {
      const float x = sum[c] * scale;
      y.v[c] = Round<O>(accumulate ? static_cast<float>(y.v[c]) + x : x);
    }
    Store<O, kVec>(at, dim - d, y);
  }
  // The end of a run of key v in chunk w.
  template <int kVec>
  __device__ __forceinline__ void Finish(unsigned v, unsigned w, int d, bool begins, bool ends, const float (&sum)[kVec]) const {
    if (v >= vocab) return;
    if (begins && ends) {
      Write<kVec>(v, d, sum);
    } else {
      Pack<float, kVec> y;
#pragma unroll
      for (int c = 0; c < kVec; ++c) y.v[c] = sum[c];
      Store<float, kVec>(parts + ((size_t)w * 2 + (begins ? 1 : 0)) * dim + d, dim - d, y);
    }
  }
};

// Zeros for the rows [block * slots, ...) that no token names.  Which these are is found from the few pairs of those rows.
template <typename T, typename O>
__device__ __forceinline__ void FillRows(const Gradient<T, O> &g, unsigned block) {
  __shared__ unsigned s_range[2], s_named[kMostSlots / 32];
  const unsigned wave = threadIdx.x >> 6;
  const unsigned v0 = block * g.slots, v1 = min(g.vocab, v0 + g.slots), slots = v1 - v0;
  if (threadIdx.x < kMostSlots / 32) s_named[threadIdx.x] = 0;
  if (wave < 2) {
    const unsigned at = WaveLowerBound(g.keys, g.m, wave == 0 ? v0 : v1);
    if ((threadIdx.x & 63u) == 0) s_range[wave] = at;
  }
  __syncthreads();
  const unsigned begin = s_range[0], end = s_range[1];
  if (end - begin <= 8 * kThreads) {
    for (unsigned p = begin + threadIdx.x; p < end; p += kThreads) {
      const unsigned k = g.keys[p] - v0;
      if (k < slots) atomicOr(&s_named[k / 32], 1u << (k % 32));
    }
  } else if (threadIdx.x < slots) {
    unsigned low = begin, high = end;
    while (low < high) {
      const unsigned mid = low + (high - low) / 2;
      if (g.keys[mid] < v0 + threadIdx.x) low = mid + 1;
      else high = mid;
    }
    if (low < end && g.keys[low] == v0 + threadIdx.x) atomicOr(&s_named[threadIdx.x / 32], 1u << (threadIdx.x % 32));
  }
  __syncthreads();
  constexpr int kVec = 16 / sizeof(O);
  const int lanes = min(64, (g.dim + kVec - 1) / kVec);  // lanes of a row
  const int groups = kThreads / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  if (group >= groups) return;
  Pack<O, kVec> zero;
#pragma unroll
  for (int c = 0; c < kVec; ++c) zero.v[c] = O(0);
  for (unsigned k = group; k < slots; k += groups) {
    if (s_named[k / 32] >> (k % 32) & 1u) continue;
    O *row = g.grad_table + (long long)(v0 + k) * g.table_stride;
    for (int d = lane * kVec; d < g.dim; d += lanes * kVec) Store<O, kVec>(row + d, g.dim - d, zero);
  }
}

// Rows of more than kNarrow elements: 2^lanes_log lanes hold kVec columns each and walk a chunk pair by pair, kAhead rows in flight.
template <typename T, typename O, int kVec>
__global__ void __launch_bounds__(kThreads) k_grad_wide(const Gradient<T, O> g) {
  if (blockIdx.x < g.fill_blocks) {
    FillRows(g, blockIdx.x);
    return;
  }
  const unsigned block = blockIdx.x - g.fill_blocks;
  const unsigned piece = block % g.pieces;
  unsigned w = ((block / g.pieces) * kThreads + threadIdx.x) >> g.lanes_log;
  if (g.lanes_log == 6) w = __builtin_amdgcn_readfirstlane(w);  // (the wave's own: keys and rows are scalar loads then)
  const int d = (int)(((piece << g.lanes_log) + (threadIdx.x & ((1u << g.lanes_log) - 1u))) * kVec);
  if (w >= g.chunks || d >= g.dim) return;
  const unsigned begin = w * g.chunk, end = min(g.m, begin + g.chunk);
  unsigned cur = g.keys[begin];
  bool begins = begin == 0 || g.keys[begin - 1] != cur;
  float sum[kVec];
#pragma unroll
  for (int c = 0; c < kVec; ++c) sum[c] = 0.0f;
  const T *column = g.grad_out + d;
  const int held = g.dim - d;
  for (unsigned p = begin; p < end; p += kAhead) {
    Pack<unsigned, kAhead> key, row;
    if (p + kAhead <= end) {
      key = *reinterpret_cast<const Pack<unsigned, kAhead> *>(g.keys + p);
      row = *reinterpret_cast<const Pack<unsigned, kAhead> *>(g.rows + p);
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {  // past the end the last key stands, without a row
        key.v[k] = g.keys[min(p + k, end - 1)];
        row.v[k] = p + k < end ? g.rows[p + k] : g.n;
      }
    }
    Pack<T, kVec> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (row.v[k] < g.n && key.v[k] < g.vocab) {
        Load<T, kVec>(column + (long long)row.v[k] * g.out_stride, held, &x[k]);
      } else {
#pragma unroll
        for (int c = 0; c < kVec; ++c) x[k].v[c] = T(0);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (key.v[k] != cur) {
        g.template Finish<kVec>(cur, w, d, begins, true, sum);
        cur = key.v[k];
        begins = true;
#pragma unroll
        for (int c = 0; c < kVec; ++c) sum[c] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < kVec; ++c) sum[c] += static_cast<float>(x[k].v[c]);
    }
  }
  g.template Finish<kVec>(cur, w, d, begins, end == g.m || g.keys[end] != cur, sum);
}

__device__ __forceinline__ float WaveSum(float v) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Rows of up to kDim <= kNarrow elements: a lane takes a pair with its whole row, a wave 64 pairs of a chunk at a time.  While the key stays
// the same the lanes add up what is theirs; when it changes they meet.
template <typename T, typename O, int kDim>
__global__ void __launch_bounds__(kThreads) k_grad_narrow(const Gradient<T, O> g) {
  if (blockIdx.x < g.fill_blocks) {
    FillRows(g, blockIdx.x);
    return;
  }
  const unsigned w = __builtin_amdgcn_readfirstlane(((blockIdx.x - g.fill_blocks) * kThreads + threadIdx.x) >> 6);
  if (w >= g.chunks) return;
  const unsigned lane = threadIdx.x & 63u;
  const unsigned begin = w * g.chunk, end = min(g.m, begin + g.chunk);
  unsigned cur = g.keys[begin];
  bool begins = begin == 0 || g.keys[begin - 1] != cur;
  float sum[kDim];
#pragma unroll
  for (int c = 0; c < kDim; ++c) sum[c] = 0.0f;
  constexpr int kRounds = 4;
  for (unsigned p = begin; p < end; p += 64 * kRounds) {
    unsigned key[kRounds];
    Pack<T, kDim> x[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const unsigned at = p + k * 64 + lane;
      key[k] = g.keys[min(at, end - 1)];
      const unsigned row = g.rows[min(at, end - 1)];
      if (at < end && row < g.n && key[k] < g.vocab) {
        Load<T, kDim>(g.grad_out + (long long)row * g.out_stride, g.dim, &x[k]);
      } else {
#pragma unroll
        for (int c = 0; c < kDim; ++c) x[k].v[c] = T(0);
      }
    }
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const bool same = key[k] == cur;
      if (__ballot(!same) == 0ull) {
#pragma unroll
        for (int c = 0; c < kDim; ++c) sum[c] += static_cast<float>(x[k].v[c]);
        continue;
      }
      // the run that came in ends here
      float total[kDim];
#pragma unroll
      for (int c = 0; c < kDim; ++c) total[c] = WaveSum(sum[c] + (same ? static_cast<float>(x[k].v[c]) : 0.0f));
      if (lane == 0) g.template Finish<kDim>(cur, w, 0, begins, true, total);
      // the last key goes on; those between are whole: sums over runs of equal keys, by steps of doubled length
      const unsigned last = __builtin_amdgcn_readlane(key[k], 63);
      const bool between = !same && key[k] != last;
      if (__ballot(between) != 0ull) {
        float run[kDim];
#pragma unroll
        for (int c = 0; c < kDim; ++c) run[c] = static_cast<float>(x[k].v[c]);
        for (int off = 1; off < 64; off <<= 1) {
          const bool joins = __shfl_up(key[k], off) == key[k] && lane >= (unsigned)off;
#pragma unroll
          for (int c = 0; c < kDim; ++c) {
            const float o = __shfl_up(run[c], off);
            if (joins) run[c] += o;
          }
        }
        const unsigned after = __shfl_down(key[k], 1);
        if (between && after != key[k]) g.template Finish<kDim>(key[k], w, 0, true, true, run);
      }
#pragma unroll
      for (int c = 0; c < kDim; ++c) sum[c] = key[k] == last ? static_cast<float>(x[k].v[c]) : 0.0f;
      cur = last;
      begins = true;
    }
  }
  float total[kDim];
#pragma unroll
  for (int c = 0; c < kDim; ++c) total[c] = WaveSum(sum[c]);
  if (lane == 0) g.template Finish<kDim>(cur, w, 0, begins, end == g.m || g.keys[end] != cur, total);
}

// Chunk w: whether a run begins in it that goes on beyond its end, and the last chunk that run reaches.
template <typename T, typename O>
__device__ __forceinline__ bool GoesOn(const Gradient<T, O> &g, unsigned w, unsigned *v, unsigned *last) {
  const unsigned begin = w * g.chunk, end = begin + g.chunk;
  if (end >= g.m) return false;
  *v = g.keys[end];
  if (*v >= g.vocab || g.keys[end - 1] != *v) return false;
  if (g.keys[begin] == *v && begin != 0 && g.keys[begin - 1] == *v) return false;
  *last = (WaveLowerBound(g.keys + end, g.m - end, *v + 1u) + end - 1u) / g.chunk;
  return true;
}

// The parts of the runs that go on, wide rows: a lane per column, the waves of a workgroup share the parts.
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) k_grad_join_wide(const Gradient<T, O> g) {
  __shared__ float s_sum[kThreads / 64][64];
  unsigned v, last;
  const unsigned w = blockIdx.x;
  if (!GoesOn(g, w, &v, &last)) return;
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  constexpr unsigned kWaves = kThreads / 64;
  for (int d0 = (int)blockIdx.y * 64; d0 < g.dim; d0 += 64 * (int)gridDim.y) {
    const int d = min(d0 + (int)lane, g.dim - 1);
    float sum[1] = {wave == 0 ? g.parts[((size_t)w * 2 + 1) * g.dim + d] : 0.0f};
#pragma unroll 8
    for (unsigned x = w + 1u + wave; x <= last; x += kWaves) sum[0] += g.parts[(size_t)x * 2 * g.dim + d];
    s_sum[wave][lane] = sum[0];
    __syncthreads();
    if (wave == 0 && d0 + (int)lane < g.dim) {
      for (unsigned k = 1; k < kWaves; ++k) sum[0] += s_sum[k][lane];
      g.template Write<1>(v, d, sum);
    }
    __syncthreads();
  }
}

// The same for narrow rows: a wave per run, its lanes share the parts.
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) k_grad_join_narrow(const Gradient<T, O> g) {
  const unsigned w = __builtin_amdgcn_readfirstlane((blockIdx.x * kThreads + threadIdx.x) >> 6), lane = threadIdx.x & 63u;
  unsigned v, last;
  if (w >= g.chunks || !GoesOn(g, w, &v, &last)) return;
  for (int d = 0; d < g.dim; ++d) {
    float sum[1] = {lane == 0 ? g.parts[((size_t)w * 2 + 1) * g.dim + d] : 0.0f};
#pragma unroll 4
    for (unsigned x = w + 1u + lane; x <= last; x += 64u) sum[0] += g.parts[(size_t)x * 2 * g.dim + d];
    sum[0] = WaveSum(sum[0]);
    if (lane == 0) g.template Write<1>(v, d, sum);
  }
}

// Pairs of a chunk.  Wide: 32, so that 32,768 pairs by 4096 columns are work for every CU, and more where the pairs
// alone fill the chip, since each chunk leaves two rows of parts.  Narrow: from 64 (a round of a wave) on, by the same rule.
unsigned ChunkOf(unsigned m, int dim) {
  const unsigned least = dim > kNarrow ? 32 : 64, most = dim > kNarrow ? 256 : 1024;
  unsigned c = least;
  while (c < most && m / c > 16384) c *= 2;
  return c;
}

// ------------------------------------------------------------------ checks

constexpr int kMostDim = (1 << 24) - 1;  // (a grid's second dimension counts 65,535 pieces of a row of 256 elements at least)

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
  if (dim < 1 || dim > kMostDim) throw std::runtime_error("bad dimension");
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
  WithType(a.type, [&](auto e) {
    WithToken(a.bags.bits, [&](auto token) {
      typedef decltype(e) T;
      constexpr int kVec = 16 / sizeof(T);
      if (a.dim >= kVec) LaunchLookup<T, kVec, decltype(token)>(a, st);
      else LaunchLookup<T, 1, decltype(token)>(a, st);
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
  if (dim < 1 || dim > kMostDim) throw std::runtime_error("bad dimension");
  const unsigned m = (unsigned)(n * bag), chunk = ChunkOf(m, dim);
  return (size_t)((m + chunk - 1) / chunk) * 2 * dim * sizeof(float);
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
  auto launch = [&](auto t, auto o) {
    typedef decltype(t) T;
    typedef decltype(o) O;
    Gradient<T, O> g;
    g.keys = a.keys;
    g.rows = a.rows;
    g.m = m;
    g.n = (unsigned)a.n;
    g.vocab = (unsigned)a.vocab;
    g.grad_out = static_cast<const T *>(a.grad_out);
    g.out_stride = a.out_stride;
    g.grad_table = static_cast<O *>(a.grad_table);
    g.table_stride = a.table_stride;
    g.dim = a.dim;
    g.scale = a.scale;
    g.accumulate = a.accumulate;
    g.chunk = ChunkOf(m, a.dim);
    g.chunks = (m + g.chunk - 1) / g.chunk;
    g.parts = static_cast<float *>(a.work);
    g.slots = (unsigned)std::min<size_t>(std::max<size_t>(65536 / (a.dim * sizeof(O)), 1), kMostSlots);
    g.fill_blocks = a.accumulate ? 0 : (unsigned)((a.vocab + g.slots - 1) / g.slots);
    g.lanes_log = 6;
    g.pieces = 1;
    if (a.dim > kNarrow) {
      constexpr int kVec = 16 / sizeof(T);
      const unsigned vectors = (unsigned)(a.dim + kVec - 1) / kVec;
      g.lanes_log = std::min(LogAtLeast(vectors), 6);
      g.pieces = (vectors + (1u << g.lanes_log) - 1) >> g.lanes_log;
      const unsigned long long blocks =
          ((((unsigned long long)g.chunks << g.lanes_log) + kThreads - 1) / kThreads) * g.pieces + g.fill_blocks;
      if (blocks >= (1ull << 31)) throw std::runtime_error("too many tokens of this width");
      if (blocks > 0) hipLaunchKernelGGL((k_grad_wide<T, O, kVec>), dim3((unsigned)blocks), dim3(kThreads), 0, st, g);
      if (g.chunks > 1)
        hipLaunchKernelGGL((k_grad_join_wide<T, O>), dim3(g.chunks, std::min((a.dim + 63) / 64, 64)), dim3(kThreads), 0, st, g);
    } else {
      const unsigned wave_blocks = (g.chunks + kThreads / 64 - 1) / (kThreads / 64), blocks = wave_blocks + g.fill_blocks;
      auto run = [&](auto width) {
        hipLaunchKernelGGL((k_grad_narrow<T, O, decltype(width)::value>), dim3(blocks), dim3(kThreads), 0, st, g);
      };
      if (blocks > 0) {
        if (a.dim == 1) run(std::integral_constant<int, 1>());
        else if (a.dim == 2) run(std::integral_constant<int, 2>());
        else if (a.dim <= 4) run(std::integral_constant<int, 4>());
        else run(std::integral_constant<int, 8>());
      }
      if (g.chunks > 1) hipLaunchKernelGGL((k_grad_join_narrow<T, O>), dim3(wave_blocks), dim3(kThreads), 0, st, g);
    }
  };
  WithType(a.type, [&](auto t) {
    if (a.table_type == kFloat32) launch(t, float());
    else launch(t, t);
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
