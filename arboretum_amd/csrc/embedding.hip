// Embedding lookup over bags of tokens and the gradient of its table by sorted tokens.
//
//   lookup    out[i]        = scale * sum_j table[token(i, j)]
//   gradient  grad_table[v] = scale * sum of grad_out[i] over all (i, j) with token(i, j) = v
//
// The gradient gathers: the (token, bag) pairs are put in order of tokens first (a radix sort), so that every sum is
// formed in an order that depends on the tokens alone, and no atomic decides it.
#include <algorithm>
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
  __device__ __forceinline__ Token At(long long i, long long j) const { return tokens[i * token_stride + j * bag_stride]; }
  // The row of the table that a token names; `vocab` for none (negative tokens are large ones without a sign).
  __device__ __forceinline__ unsigned Row(Token t) const {
    typedef std::make_unsigned_t<Token> Word;
    return (unsigned)min((Word)t, (Word)vocab);
  }
  __device__ __forceinline__ bool Wrong(Token t) const { return t != -1 && Row(t) == vocab; }
  // (a branch that a call without a status word passes by)
  template <int kTokens>
  __device__ __forceinline__ void Report(const Token (&t)[kTokens]) const {
    if (status == nullptr) return;
    bool wrong = false;
#pragma unroll
    for (int k = 0; k < kTokens; ++k) wrong = wrong || Wrong(t[k]);
    if (wrong) *status = 1u;
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

// Bags of one token: rows are copied, scaled.  2^lanes_log lanes take a piece of kPieces vectors a lane of a row, so
// that all its loads are in flight at once (blockIdx.y: which piece).  Here and below the last vector of a row that
// is not whole vectors wide is moved back to end with the row: two lanes then write the same values to the same
// place.
constexpr int kPieces = 4;
template <typename T, int kVec, bool kPast, typename Token>
__global__ void __launch_bounds__(kThreads) k_embedding_one(const Bags<Token> bags, const Rows<T> r, int lanes_log) {
  const long long i = (long long)(((unsigned long long)blockIdx.x * kThreads + threadIdx.x) >> lanes_log);
  if (i >= bags.n) return;
  const unsigned lane = threadIdx.x & ((1u << lanes_log) - 1u);
  const int step = kVec << lanes_log;
  const int first = (int)blockIdx.y * (step * kPieces) + (int)lane * kVec;
  const Token token[1] = {bags.At(i, 0)};
  const unsigned t = bags.Row(token[0]);
  if (blockIdx.y == 0 && lane == 0) bags.Report(token);
  const T *from = r.table + (long long)min(t, bags.vocab - 1u) * r.table_stride;
  T *to = r.out + i * r.out_stride;
  Pack<T, kVec> x[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) x[k] = *reinterpret_cast<const Pack<T, kVec> *>(from + min(first + k * step, r.dim - kVec));
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
#pragma unroll
    for (int c = 0; c < kVec; ++c) x[k].v[c] = t < bags.vocab ? Round<T>(static_cast<float>(x[k].v[c]) * r.scale) : T(0);
    if (first + k * step >= r.dim) continue;
    T *at = to + min(first + k * step, r.dim - kVec);
    if (kPast) StorePast<T, kVec>(at, x[k]);
    else *reinterpret_cast<Pack<T, kVec> *>(at) = x[k];
  }
}

// Bags of several tokens.  A row of the result is 2^lanes_log lanes wide (kVec elements a lane), and 2^shares_log
// shares of them take every so many-th token each and meet in the end, by steps of halves.  kAhead tokens of a lane
// are in flight; where there is no token the last row of the table is read and not added.  All eight are summed before
// they join the sum of those before them: no more additions than one after the other, and an eighth of a chain's
// error.  (Rows of 16 bits, eight elements a lane, four at a time: eight take 89 registers for 63 and 2 % of the time,
// and the result is rounded to 2^-8 or 2^-11.)
constexpr int kAhead = 8;
__device__ __forceinline__ float SumOfFour(const float (&x)[4]) { return (x[0] + x[1]) + (x[2] + x[3]); }
template <typename T, int kVec, typename Token>
__global__ void __launch_bounds__(kThreads)
k_embedding_bag(const Bags<Token> bags, const Rows<T> r, int lanes_log, int shares_log) {
  const long long i = (long long)(((unsigned long long)blockIdx.x * kThreads + threadIdx.x) >> (lanes_log + shares_log));
  const bool live = i < bags.n;
  const unsigned lane = threadIdx.x & ((1u << lanes_log) - 1u);
  const unsigned share = (threadIdx.x >> lanes_log) & ((1u << shares_log) - 1u), shares = 1u << shares_log;
  const int column = ((int)blockIdx.y << lanes_log) * kVec + (int)lane * kVec, d = min(column, r.dim - kVec);
  constexpr bool kEights = sizeof(T) == 4;
  float sum[kVec];
#pragma unroll
  for (int c = 0; c < kVec; ++c) sum[c] = 0.0f;
  if (live && column < r.dim) {
    const Token *at = bags.tokens + i * bags.token_stride;
    const T *table = r.table + d;
    auto add = [&](const Token (&token)[kAhead]) {
      Pack<T, kVec> x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        x[k] = *reinterpret_cast<const Pack<T, kVec> *>(table + (long long)min(bags.Row(token[k]), bags.vocab - 1u) * r.table_stride);
#pragma unroll
      for (int c = 0; c < kVec; ++c) {
        float part = kEights ? 0.0f : sum[c];
#pragma unroll
        for (int h = 0; h < kAhead; h += 4) {
          float y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = bags.Row(token[h + k]) < bags.vocab ? static_cast<float>(x[h + k].v[c]) : 0.0f;
          part = kEights && h == 0 ? SumOfFour(y) : part + SumOfFour(y);
        }
        sum[c] = kEights ? sum[c] + part : part;
      }
      if (blockIdx.y == 0 && lane == 0) bags.Report(token);
    };
    const unsigned bag = (unsigned)bags.bag;
    Token token[kAhead];
    unsigned j = share;
    for (; j + (kAhead - 1) * shares < bag; j += kAhead * shares) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) token[k] = at[(j + k * shares) * bags.bag_stride];
      add(token);
    }
    if (j < bag) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) token[k] = j + k * shares < bag ? at[(j + k * shares) * bags.bag_stride] : Token(-1);
      add(token);
    }
  }
  for (int s = shares_log - 1; s >= 0; --s)
#pragma unroll
    for (int c = 0; c < kVec; ++c) sum[c] += __shfl_xor(sum[c], 1 << (lanes_log + s));
  if (live && share == 0 && column < r.dim) {
    Pack<T, kVec> y;
#pragma unroll
    for (int c = 0; c < kVec; ++c) y.v[c] = Round<T>(sum[c] * r.scale);
    *reinterpret_cast<Pack<T, kVec> *>(r.out + i * r.out_stride + d) = y;
  }
}

// Rows of one element over so many bags that their tokens, column by column (the leaves of trees), come from memory
// and not from the last-level cache of 256 MB.  A thread takes four neighbouring bags, whose tokens are one load, and
// the tokens of the next columns are in flight while these are looked up.  Reading the tokens alone takes 135 us for
// a million bags of 200; the rest is the lookups.  (With the pieces of the table that a column names copied to the
// LDS first 290 and more: finding the pieces takes longer than the LDS saves.)
// Taken from 512 MB of tokens on, where there are two workgroups for a CU.  Us with a bag a thread / here, 256 leaves
// a column: tokens of 32 bits, 256 MB: 3,355,446 x 20 71 / 67, 671,091 x 100 75 / 76, 335,547 x 200 80 / 108; 512 MB:
// 158 / 146, 177 / 162, 671,091 x 200 187 / 166, 335,547 x 400 206 / 233; 1 GB: 316 / 282, 350 / 289, 355 / 317.  Of
// 64 bits, 256 MB: 53 / 49, 56 / 63, 54 / 84; 512 MB: 126 / 113, 133 / 117, 335,547 x 200 140 / 145; 1 GB: 252 / 223,
// 251 / 225, 260 / 230.  A table that the L1 holds, or one whose rows are named all over, makes less of it: 512 MB of
// 32 bits over 100 x 64 leaves 138 / 149, bags of three out of 200,000 514 / 542.
constexpr int kColumns = 4;  // (SumOfFour)
constexpr int kBagsOfThread = 4;
constexpr int kColumnBags = kThreads * kBagsOfThread;
constexpr long long kManyTokenBytes = 1ll << 29;
constexpr long long kManyBags = 2 * 256 * kColumnBags;

template <typename T, typename Token>
__global__ void __launch_bounds__(kThreads) k_embedding_columns(const Bags<Token> bags, const Rows<T> r) {
  const long long first = (long long)blockIdx.x * kColumnBags + threadIdx.x * kBagsOfThread;
  const int held = (int)max(0ll, min((long long)kBagsOfThread, bags.n - first));
  Token next[kColumns][kBagsOfThread];
  auto fetch = [&](int j) {
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      const Token *at = bags.tokens + min(j + c, bags.bag - 1) * bags.bag_stride + first;
      if (held == kBagsOfThread) {
        *reinterpret_cast<Pack<Token, kBagsOfThread> *>(next[c]) = *reinterpret_cast<const Pack<Token, kBagsOfThread> *>(at);
      } else {
#pragma unroll
        for (int k = 0; k < kBagsOfThread; ++k) next[c][k] = k < held ? at[k] : Token(-1);
      }
#pragma unroll
      for (int k = 0; k < kBagsOfThread; ++k)
        if (j + c >= bags.bag) next[c][k] = Token(-1);
    }
  };
  float sum[kBagsOfThread] = {}, part[kBagsOfThread] = {};  // of the columns before, of up to sixteen since
  fetch(0);
  for (int j = 0; j < bags.bag; j += kColumns) {
    unsigned t[kColumns][kBagsOfThread];
    float x[kColumns][kBagsOfThread];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      bags.Report(next[c]);
#pragma unroll
      for (int k = 0; k < kBagsOfThread; ++k) t[c][k] = bags.Row(next[c][k]);
    }
    if (j + kColumns < bags.bag) fetch(j + kColumns);
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int k = 0; k < kBagsOfThread; ++k)
        x[c][k] = static_cast<float>(r.table[(long long)min(t[c][k], bags.vocab - 1u) * r.table_stride]);
#pragma unroll
    for (int k = 0; k < kBagsOfThread; ++k) {
      float y[kColumns];
#pragma unroll
      for (int c = 0; c < kColumns; ++c) y[c] = t[c][k] < bags.vocab ? x[c][k] : 0.0f;
      part[k] += SumOfFour(y);
    }
    if ((j / kColumns) % 4 == 3) {
#pragma unroll
      for (int k = 0; k < kBagsOfThread; ++k) {
        sum[k] += part[k];
        part[k] = 0.0f;
      }
    }
  }
  for (int k = 0; k < held; ++k) r.out[(first + k) * r.out_stride] = Round<T>((sum[k] + part[k]) * r.scale);
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
  const bool past = (size_t)a.bags.n * a.dim * sizeof(T) > kStreamedBytes;
  if constexpr (kVec == 1) {
    if (a.dim == 1 && a.bags.bag > 1 && a.bags.token_stride == 1 && a.bags.bag_stride > 1 && a.bags.n >= kManyBags &&
        a.bags.n * a.bags.bag * (long long)sizeof(Token) >= kManyTokenBytes) {
      const unsigned blocks = (unsigned)((a.bags.n + kColumnBags - 1) / kColumnBags);
      hipLaunchKernelGGL((k_embedding_columns<T, Token>), dim3(blocks), dim3(kThreads), 0, st, bags, r);
      return;
    }
  }
  const long long vectors = (a.dim + kVec - 1) / kVec;
  const int lanes_log = std::min(LogAtLeast(vectors), 6);
  long long per_row = (vectors + (1ll << lanes_log) - 1) >> lanes_log;  // pieces of a row
  int group_log = lanes_log, shares_log = 0;
  if (a.bags.bag == 1) {
    per_row = (per_row + kPieces - 1) / kPieces;
  } else {
    // Where the tokens of a bag lie beside each other the lanes of a wave read along them; otherwise they read along the
    // bags, unless these do not fill the chip (4 waves a CU).
    const int most = std::min(6 - lanes_log, LogAtLeast((a.bags.bag + 31) / 32));
    if (a.bags.bag_stride <= a.bags.token_stride) shares_log = most;
    else
      while (shares_log < most && ((a.bags.n * per_row) << (lanes_log + shares_log)) < 65536) ++shares_log;
    group_log += shares_log;
  }
  // (a launch counts its threads with 32 bits)
  const long long most = (1ll << 31) >> group_log;
  for (long long i = 0; i < a.bags.n; i += most) {
    Bags<Token> some = bags;
    some.n = std::min(most, a.bags.n - i);
    if (some.tokens) some.tokens += i * some.token_stride;
    Rows<T> to = r;
    to.out += i * r.out_stride;
    const dim3 grid((unsigned)(((some.n << group_log) + kThreads - 1) / kThreads), (unsigned)per_row);
    const dim3 block(kThreads);
    if (a.bags.bag != 1) hipLaunchKernelGGL((k_embedding_bag<T, kVec, Token>), grid, block, 0, st, some, to, lanes_log, shares_log);
    else if (past) hipLaunchKernelGGL((k_embedding_one<T, kVec, true, Token>), grid, block, 0, st, some, to, lanes_log);
    else hipLaunchKernelGGL((k_embedding_one<T, kVec, false, Token>), grid, block, 0, st, some, to, lanes_log);
  }
}

// -------------------------------------------------------------------- sort

// Division of numbers below 2^31 by a number that stays the same (Granlund and Montgomery, "Division by invariant
// integers using multiplication"): with 2^(l-1) < d <= 2^l, factor = floor(2^(31+l) / d) + 1 makes p factor /
// 2^(31+l) exceed p / d by less than 1 / d.
struct Divider {
  unsigned by, factor;
  int shift;
  explicit Divider(unsigned d) : by(d), factor(0), shift(0) {
    if (d < 2) return;  // (factor 0)
    int l = 1;
    while ((1ull << l) < d) ++l;
    factor = (unsigned)((1ull << (31 + l)) / d + 1);
    shift = l - 1;
  }
  __device__ __forceinline__ unsigned Quotient(unsigned p) const { return factor == 0 ? p : __umulhi(p, factor) >> shift; }
};

// The pairs of a call, numbered in the order the tokens lie in memory.
template <typename Token>
struct Pairs {
  Bags<Token> bags;
  unsigned m;
  bool by_column;  // pair p is token p / n of bag p % n, else token p % bag of bag p / bag
  bool flat;       // ... and stands at tokens[p]
  Divider line;    // n or bag
  __device__ __forceinline__ unsigned Bag(unsigned p) const {
    const unsigned q = line.Quotient(p);
    return by_column ? p - q * line.by : q;
  }
  // Tokens of the pairs first, first + step, ... ; past the last pair that one's.
  template <int kTokens>
  __device__ __forceinline__ void Get(unsigned first, unsigned step, Token (&to)[kTokens]) const {
    if (flat) {
#pragma unroll
      for (int k = 0; k < kTokens; ++k) to[k] = bags.tokens[min(first + k * step, m - 1)];
    } else {
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        const unsigned p = min(first + k * step, m - 1), q = line.Quotient(p), rest = p - q * line.by;
        to[k] = bags.At(by_column ? rest : q, by_column ? q : rest);
      }
    }
  }
};

template <typename Token>
Pairs<Token> PairsOf(const TokenBags &b, unsigned m) {
  const bool by_column = b.token_stride < b.bag_stride;
  const bool flat = by_column ? (b.token_stride == 1 || b.n == 1) && (b.bag_stride == b.n || b.bag == 1)
                              : (b.bag_stride == 1 || b.bag == 1) && (b.token_stride == b.bag || b.n == 1);
  return Pairs<Token>{BagsOf<Token>(b), m, by_column, flat, Divider(by_column ? (unsigned)b.n : (unsigned)b.bag)};
}

// Lanes of the wave that hold the same digit as this one, for kSome digits a lane: low and high come in as the lanes that
// hold a digit at all.
template <int kSome>
__device__ __forceinline__ void DigitPeers(const unsigned (&d)[kSome], int bits, unsigned (&low)[kSome], unsigned (&high)[kSome]) {
  for (int b = 0; b < bits; ++b) {
#pragma unroll
    for (int k = 0; k < kSome; ++k) {
      const int set = __builtin_amdgcn_sbfe((int)d[k], b, 1);  // -1 or 0
      const unsigned long long m = __ballot(set != 0);
      low[k] &= ~((unsigned)m ^ (unsigned)set);
      high[k] &= ~((unsigned)(m >> 32) ^ (unsigned)set);
    }
  }
}

// Lanes below this one in a mask.
__device__ __forceinline__ unsigned LanesBelow(unsigned low, unsigned high) {
  return __builtin_amdgcn_mbcnt_hi(high, __builtin_amdgcn_mbcnt_lo(low, 0u));
}

// ---- few pairs: one launch
//
// Every workgroup has a range of the vocabulary.  It reads all tokens (they come out of the L2), counts those below
// its range, which is where its pairs start in the result, keeps those within, and sorts them in the LDS.  Nothing
// passes between workgroups.

constexpr int kRangeThreads = 1024;
constexpr int kRangeWaves = kRangeThreads / 64;
constexpr int kRangeBits = 8;  // of a digit, at most
constexpr unsigned kMostRangePairs = 32768;
constexpr unsigned kMostRanges = 256;  // a workgroup per CU

// Pairs are kept as (key - first key of the range) << place_bits | place.  All rounds are unrolled, each behind its
// own test: with 32 of them 193 scalar registers are spilled into vector registers, and with tokens of 64 bits, which
// are all in flight at once, 6 vector registers to scratch memory (32,768 pairs: 19.3 us, 21.2 with 64 bits).
template <int kRounds, typename Token>
__global__ void __launch_bounds__(kRangeThreads)
k_sort_ranges(const Pairs<Token> in, unsigned span, int key_bits, int place_bits, unsigned *__restrict__ keys,
              unsigned *__restrict__ rows) {
  __shared__ unsigned s_pair[kRounds * kRangeThreads];
  constexpr int kCounters = kRangeWaves << kRangeBits, kOwn = kCounters / kRangeThreads;
  __shared__ __align__(16) unsigned s_count[kCounters];  // pairs of a digit, then their place; the waves of a digit beside each other
  __shared__ unsigned s_sum[2][kRangeWaves];
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned v0 = blockIdx.x * span;
  if (v0 > in.bags.vocab) return;
  const unsigned here = min(span, in.bags.vocab + 1u - v0);  // keys of the range (a key less v0 wraps to a large one below it)
  Token token[kRounds];
  unsigned key[kRounds];
  in.Get(threadIdx.x, kRangeThreads, token);
#pragma unroll
  for (int k = 0; k < kRounds; ++k) key[k] = k * kRangeThreads + threadIdx.x < in.m ? in.bags.Row(token[k]) : ~0u;
  if (blockIdx.x == 0) in.bags.Report(token);
  unsigned within = 0, below = 0;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    within += (unsigned)__popcll(__ballot(key[k] - v0 < here));
    below += (unsigned)__popcll(__ballot(key[k] < v0));
  }
  if (lane == 0) {
    s_sum[0][wave] = within;
    s_sum[1][wave] = below;
  }
  __syncthreads();
  unsigned at = 0, held = 0, start = 0;
#pragma unroll
  for (unsigned w = 0; w < kRangeWaves; ++w) {
    if (w < wave) at += s_sum[0][w];
    held += s_sum[0][w];
    start += s_sum[1][w];
  }
  if (held == 0) return;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool mine = key[k] - v0 < here;
    const unsigned long long all = __ballot(mine);
    const unsigned to = at + LanesBelow((unsigned)all, (unsigned)(all >> 32));
    if (mine) s_pair[to] = (key[k] - v0) << place_bits | (k * kRangeThreads + threadIdx.x);
    at += (unsigned)__popcll(all);
  }
  const int passes = (key_bits + kRangeBits - 1) / kRangeBits;
  // a wave's pairs are a run of them: `rounds` times 64
  const unsigned rounds = (held + kRangeThreads - 1) / kRangeThreads, first = wave * rounds * 64u;
  for (int pass = 0; pass < passes; ++pass) {
    const int bits = (key_bits + passes - 1) / passes, shift = place_bits + pass * bits;
    unsigned pair[kRounds], place[kRounds];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) s_count[k * kRangeThreads + threadIdx.x] = 0;
    __syncthreads();  // (the pairs are in place, too)
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (k < (int)rounds) {
        const unsigned i = first + k * 64u + lane;
        const bool valid = i < held;
        pair[k] = valid ? s_pair[i] : 0u;
        const unsigned d[1] = {(pair[k] >> shift) & ((1u << bits) - 1u)};
        const unsigned long long all = __ballot(valid);
        unsigned low[1] = {(unsigned)all}, high[1] = {(unsigned)(all >> 32)};
        DigitPeers(d, bits, low, high);
        const unsigned less = LanesBelow(low[0], high[0]);
        unsigned *count = &s_count[d[0] * kRangeWaves + wave];
        const unsigned before = *count;
        place[k] = before + less;
        __builtin_amdgcn_wave_barrier();  // every lane has read its counter
        if (valid && less == 0) *count = before + __popc(low[0]) + __popc(high[0]);
        __builtin_amdgcn_wave_barrier();
      }
    }
    __syncthreads();
    // exclusive sum over (digit, wave), kOwn counters a thread
    unsigned own[kOwn], mine = 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      own[k] = s_count[threadIdx.x * kOwn + k];
      mine += own[k];
    }
    unsigned sum = mine;
    for (int off = 1; off < 64; off <<= 1) {
      const unsigned o = __shfl_up(sum, off);
      if (lane >= (unsigned)off) sum += o;
    }
    if (lane == 63) s_sum[0][wave] = sum;
    __syncthreads();
    for (unsigned w = 0; w < wave; ++w) sum += s_sum[0][w];
    sum -= mine;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      s_count[threadIdx.x * kOwn + k] = sum;
      sum += own[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      if (k < (int)rounds && first + k * 64u + lane < held) {
        const unsigned d = (pair[k] >> shift) & ((1u << bits) - 1u);
        s_pair[s_count[d * kRangeWaves + wave] + place[k]] = pair[k];
      }
    }
    __syncthreads();
  }
  if (passes == 0) __syncthreads();
  for (unsigned i = threadIdx.x; i < held; i += kRangeThreads) {
    const unsigned pair = s_pair[i], p = pair & ((1u << place_bits) - 1u);
    keys[start + i] = v0 + (pair >> place_bits);
    rows[start + i] = in.Bag(p);
  }
}

// ---- many pairs: least significant digit first
//
// Up to 9 bits a pass (two passes up to a vocabulary of 262,143), four launches each, and two where 32 tiles hold all
// pairs.  A tile of up to 8192 pairs is put in order in the LDS, so that the pairs of a digit leave as one run.

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kSortRounds = 8, kFewestRounds = 2;  // pairs per thread
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr unsigned kXcds = 8;
constexpr unsigned kGroupTiles = 32;  // tiles whose counts are summed up by one workgroup

// Where a pass takes its pairs from: the tokens themselves, or the keys and rows of the pass before.
template <typename Token>
struct FromTokens {
  Pairs<Token> pairs;
  unsigned m;
  typedef Token Raw;
  template <int kSome>
  __device__ __forceinline__ void Get(unsigned first, unsigned step, Token (&to)[kSome]) const {
    pairs.Get(first, step, to);
  }
  // kSome pairs side by side
  template <int kSome>
  __device__ __forceinline__ void Beside(unsigned p, Token (&to)[kSome]) const {
    typedef Pack<Token, kSome> Some;
    if (pairs.flat && p + kSome <= m) *reinterpret_cast<Some *>(to) = *reinterpret_cast<const Some *>(pairs.bags.tokens + p);
    else pairs.Get(p, 1, to);
  }
  template <int kSome>
  __device__ __forceinline__ void Report(const Token (&t)[kSome]) const {
    pairs.bags.Report(t);
  }
  __device__ __forceinline__ unsigned Key(Token t) const { return pairs.bags.Row(t); }
  __device__ __forceinline__ unsigned Row(unsigned p) const { return pairs.Bag(p); }
};
struct FromPairs {
  const unsigned *keys, *rows;
  unsigned m;
  typedef unsigned Raw;
  template <int kSome>
  __device__ __forceinline__ void Get(unsigned first, unsigned step, unsigned (&to)[kSome]) const {
#pragma unroll
    for (int k = 0; k < kSome; ++k) to[k] = keys[min(first + k * step, m - 1)];
  }
  template <int kSome>
  __device__ __forceinline__ void Beside(unsigned p, unsigned (&to)[kSome]) const {
    if (p + kSome <= m) *reinterpret_cast<Pack<unsigned, kSome> *>(to) = *reinterpret_cast<const Pack<unsigned, kSome> *>(keys + p);
    else Get(p, 1, to);
  }
  template <int kSome>
  __device__ __forceinline__ void Report(const unsigned (&)[kSome]) const {}
  __device__ __forceinline__ unsigned Key(unsigned key) const { return key; }
  __device__ __forceinline__ unsigned Row(unsigned p) const { return rows[p]; }
};

struct Digit {
  int shift, bits;
  unsigned mask;
  __device__ __forceinline__ unsigned Of(unsigned key) const { return __builtin_amdgcn_ubfe(key, shift, bits); }
};

// Digit counts of one tile (kPairs pairs a thread): counts[tile * kDigits + digit].  A thread's pairs lie beside each
// other and equal neighbours are counted as one, and a wave of one digit only as one: pairs that are nearly in order
// (leaves, tree by tree; the last pass) would otherwise queue for one counter of the LDS.
template <int kPairs, typename Source>
__global__ void __launch_bounds__(kSortThreads) k_sort_count(const Source in, const Digit digit, unsigned *__restrict__ counts) {
  constexpr int kBeside = kPairs < 4 ? kPairs : 4, kRounds = kPairs / kBeside;
  __shared__ unsigned s_count[kDigits];
  const unsigned tile = blockIdx.x;
  if (threadIdx.x < kDigits) s_count[threadIdx.x] = 0;
  __syncthreads();
  const unsigned base = tile * (kSortThreads * kPairs) + threadIdx.x * kBeside;
  typename Source::Raw raw[kRounds][kBeside];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) in.Beside(base + r * kSortThreads * kBeside, raw[r]);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) in.Report(raw[r]);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const unsigned p = base + r * kSortThreads * kBeside;
    unsigned d[kBeside + 1];
#pragma unroll
    for (int k = 0; k < kBeside; ++k) d[k] = p + k < in.m ? digit.Of(in.Key(raw[r][k])) : kDigits;
    d[kBeside] = kDigits + 1;
    const unsigned one = __builtin_amdgcn_readfirstlane(d[0]);
    bool other = false;
#pragma unroll
    for (int k = 0; k < kBeside; ++k) other |= d[k] != one;
    if (__ballot(other) == 0ull) {
      if ((threadIdx.x & 63u) == 0 && one < kDigits) atomicAdd(&s_count[one], 64u * kBeside);
      continue;
    }
    unsigned run = 0;
#pragma unroll
    for (int k = 0; k < kBeside; ++k) {
      ++run;
      if (d[k + 1] != d[k]) {
        if (d[k] < kDigits) atomicAdd(&s_count[d[k]], run);
        run = 0;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x <= digit.mask) counts[(size_t)tile * kDigits + threadIdx.x] = s_count[threadIdx.x];
}

// Exclusive sums over the tiles of a group, in place, and the group's totals.  A thread per digit.
__global__ void __launch_bounds__(kDigits) k_sort_sum_tiles(unsigned *__restrict__ counts, unsigned tiles, unsigned *__restrict__ groups) {
  unsigned *v = counts + (size_t)blockIdx.x * kGroupTiles * kDigits + threadIdx.x;
  const unsigned held = min(kGroupTiles, tiles - blockIdx.x * kGroupTiles);
  unsigned c[kGroupTiles];
#pragma unroll
  for (unsigned k = 0; k < kGroupTiles; ++k) c[k] = k < held ? v[k * kDigits] : 0u;
  unsigned sum = 0;
#pragma unroll
  for (unsigned k = 0; k < kGroupTiles; ++k) {
    if (k < held) v[k * kDigits] = sum;
    sum += c[k];
  }
  groups[(size_t)blockIdx.x * kDigits + threadIdx.x] = sum;
}

// The same over groups, and the totals of all behind them.  64 digits a workgroup, its waves share the groups.
__global__ void __launch_bounds__(1024) k_sort_sum_groups(unsigned *__restrict__ groups, unsigned count) {
  __shared__ unsigned s_sum[16][64];
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, digit = blockIdx.x * 64 + lane;
  const unsigned per = (count + 15) / 16, b = min(count, wave * per), e = min(count, b + per);
  unsigned sum = 0;
#pragma unroll 8
  for (unsigned i = b; i < e; ++i) sum += groups[(size_t)i * kDigits + digit];
  s_sum[wave][lane] = sum;
  __syncthreads();
  unsigned run = 0, total = 0;
#pragma unroll
  for (unsigned w = 0; w < 16; ++w) {
    if (w < wave) run += s_sum[w][lane];
    total += s_sum[w][lane];
  }
#pragma unroll 8
  for (unsigned i = b; i < e; ++i) {
    const unsigned c = groups[(size_t)i * kDigits + digit];
    groups[(size_t)i * kDigits + digit] = run;
    run += c;
  }
  if (wave == 0) groups[(size_t)count * kDigits + digit] = total;
}

// Stable scatter of one tile of kPairs pairs a thread.  counts, groups: pairs of the same digit in the tiles of the
// group before, in the groups before; totals: pairs of each digit.  kFew: a single group, counts are those of each
// tile, and every workgroup sums them up for itself.
template <int kPairs, bool kFew, typename Source>
__global__ void __launch_bounds__(kSortThreads, kFew ? 4 : 8)  // (8 waves a SIMD: two workgroups on a CU)
k_sort_scatter(const Source in, const Digit digit, unsigned tiles, const unsigned *__restrict__ counts, const unsigned *__restrict__ groups,
               const unsigned *__restrict__ totals, unsigned *__restrict__ keys, unsigned *__restrict__ rows) {
  constexpr unsigned kSortTile = kSortThreads * kPairs, kWavePairs = kPairs * 64;
  __shared__ unsigned s_pair[kSortTile];                  // the keys, then the rows
  __shared__ unsigned short s_wave[kSortWaves][kDigits];  // pairs of each digit of a wave; then those of the waves before
  __shared__ unsigned s_first[kDigits];                   // place in the tile of the first pair of each digit
  __shared__ unsigned s_out[kDigits];                     // output position of that pair
  __shared__ unsigned s_sum[2][kDigits / 64];
  const unsigned lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  // Workgroups are dealt to the eight XCDs in turn.  Tiles that follow each other, whose runs of a digit meet inside
  // a line of memory, go to the same one (50 M pairs: 214 -> 199 us).
  const unsigned tile = kFew ? blockIdx.x : blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds;
  if (tile >= tiles) return;
  const unsigned base = tile * kSortTile, held = min(kSortTile, in.m - base);
  for (int i = threadIdx.x; i < kSortWaves * kDigits / 2; i += kSortThreads) reinterpret_cast<unsigned *>(s_wave)[i] = 0;
  typename Source::Raw raw[kPairs];
  unsigned key[kPairs], place[kPairs];
  in.Get(base + wave * kWavePairs + lane, 64, raw);
#pragma unroll
  for (int k = 0; k < kPairs; ++k) key[k] = in.Key(raw[k]);  // (past the end: the last one's, which goes nowhere)
  unsigned total = 0, before = 0;
  if (threadIdx.x <= digit.mask) {
    if (kFew) {
      unsigned c[kGroupTiles];
#pragma unroll
      for (unsigned k = 0; k < kGroupTiles; ++k) c[k] = counts[min(k, tiles - 1) * kDigits + threadIdx.x];
#pragma unroll
      for (unsigned k = 0; k < kGroupTiles; ++k) {
        total += k < tiles ? c[k] : 0u;
        before += k < tile ? c[k] : 0u;
      }
    } else {
      total = totals[threadIdx.x];
      before = counts[(size_t)tile * kDigits + threadIdx.x] + groups[(size_t)(tile / kGroupTiles) * kDigits + threadIdx.x];
    }
  }
  __syncthreads();
  {
    unsigned d[kPairs], low[kPairs], high[kPairs];
    bool other = false;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const bool valid = wave * kWavePairs + k * 64 + lane < held;
      const unsigned long long all = __ballot(valid);
      low[k] = (unsigned)all;
      high[k] = (unsigned)(all >> 32);
      d[k] = digit.Of(key[k]);
      other |= d[k] != (unsigned)__builtin_amdgcn_readfirstlane(d[k]);
    }
    if (__ballot(other) != 0ull) DigitPeers(d, digit.bits, low, high);  // (the last pass finds most waves in order: one digit)
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const bool valid = wave * kWavePairs + k * 64 + lane < held;
      const unsigned less = LanesBelow(low[k], high[k]);
      const unsigned held_of = s_wave[wave][d[k]];
      place[k] = held_of + less;
      __builtin_amdgcn_wave_barrier();  // every lane has read its counter
      if (valid && less == 0) s_wave[wave][d[k]] = (unsigned short)(held_of + __popc(low[k]) + __popc(high[k]));
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
  // thread = digit: pairs of smaller digits in the tile, and in all
  unsigned mine = 0;
  if (threadIdx.x < kDigits) {
    for (int w = 0; w < kSortWaves; ++w) {
      const unsigned c = s_wave[w][threadIdx.x];
      s_wave[w][threadIdx.x] = (unsigned short)mine;
      mine += c;
    }
  }
  unsigned in_tile = mine, in_all = total;
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned a = __shfl_up(in_tile, off), b = __shfl_up(in_all, off);
    if (lane >= (unsigned)off) {
      in_tile += a;
      in_all += b;
    }
  }
  if (lane == 63 && wave < kDigits / 64) {
    s_sum[0][wave] = in_tile;
    s_sum[1][wave] = in_all;
  }
  __syncthreads();
  if (threadIdx.x < kDigits) {
    for (unsigned w = 0; w < wave; ++w) {
      in_tile += s_sum[0][w];
      in_all += s_sum[1][w];
    }
    s_first[threadIdx.x] = in_tile - mine;
    s_out[threadIdx.x] = in_all - total + before;
  }
  __syncthreads();
  // From here on what stands past the end goes along, behind the pairs, up to the stores: no access of the LDS
  // stands behind a branch.
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    const unsigned i = wave * kWavePairs + k * 64 + lane, d = digit.Of(key[k]);
    const unsigned to = place[k] + s_first[d] + s_wave[wave][d];
    place[k] = i < held ? to : i;
  }
#pragma unroll
  for (int k = 0; k < kPairs; ++k) s_pair[place[k]] = key[k];
  __syncthreads();
  unsigned to[kPairs];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) key[k] = s_pair[k * kSortThreads + threadIdx.x];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) {
    const unsigned d = digit.Of(key[k]);
    to[k] = s_out[d] - s_first[d] + k * kSortThreads + threadIdx.x;
  }
#pragma unroll
  for (int k = 0; k < kPairs; ++k)
    if (k * kSortThreads + threadIdx.x < held) keys[to[k]] = key[k];
  __syncthreads();
  unsigned again = base + wave * kWavePairs + lane;
  asm volatile("" : "+v"(again));  // worked out anew: kept from the first loads on, the eight places would spill
#pragma unroll
  for (int k = 0; k < kPairs; ++k) key[k] = in.Row(min(again + k * 64, in.m - 1));
#pragma unroll
  for (int k = 0; k < kPairs; ++k) s_pair[place[k]] = key[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPairs; ++k) key[k] = s_pair[k * kSortThreads + threadIdx.x];
#pragma unroll
  for (int k = 0; k < kPairs; ++k)
    if (k * kSortThreads + threadIdx.x < held) rows[to[k]] = key[k];
}

int BitsOf(unsigned long long v) {
  int bits = 0;
  while (v >> bits) ++bits;
  return bits;
}

// Which way a call goes, for keys in [0, vocab].
struct SortPlan {
  unsigned m;
  // one launch: workgroups, keys of each, bits of a key within its range and of a pair's place; 0 workgroups: many pairs
  unsigned ranges, span;
  int key_bits, place_bits;
  int passes, bits;  // many pairs
  int pairs;         // of a thread
  unsigned tiles, groups;
  size_t counts_bytes, groups_bytes, pairs_bytes, bytes;
};
constexpr size_t Align256(size_t v) { return (v + 255) / 256 * 256; }

SortPlan PlanSort(long long n, int bag, long long vocab) {
  SortPlan s = {};
  s.bytes = 256;  // (so that nobody allocates nothing)
  s.m = (unsigned)(n * bag);
  if (s.m == 0) return s;
  if (s.m <= kMostRangePairs) {
    // 256 keys a workgroup are one pass; where there are fewer keys than that for so many pairs, 256 pairs a workgroup
    const long long wanted = std::max<long long>(vocab / 256 + 1, s.m / 256);
    s.ranges = (unsigned)std::min({wanted, vocab + 1, (long long)kMostRanges});
    s.span = (unsigned)(vocab / s.ranges + 1);
    s.key_bits = BitsOf(s.span - 1);
    s.place_bits = BitsOf(s.m - 1);
    if (s.key_bits + s.place_bits <= 32) return s;
    s.ranges = 0;
  }
  const int bits = BitsOf((unsigned long long)vocab);
  s.passes = (bits + kDigitBits - 1) / kDigitBits;
  s.bits = (bits + s.passes - 1) / s.passes;
  // small tiles, as long as they stay one group: a tile's work is one thing after the other (38,252 pairs, two passes:
  // 37 us with tiles of 8192 and the sums in a launch of their own, 20 with tiles of 2048 that take the sums themselves)
  s.pairs = kSortRounds;
  while (s.pairs > kFewestRounds && s.m <= s.pairs / 2 * kSortThreads * kGroupTiles) s.pairs /= 2;
  const unsigned tile = s.pairs * kSortThreads;
  s.tiles = (s.m + tile - 1) / tile;
  s.groups = (s.tiles + kGroupTiles - 1) / kGroupTiles;
  s.counts_bytes = Align256((size_t)s.tiles * kDigits * sizeof(unsigned));
  s.groups_bytes = (size_t)(s.groups + 1) * kDigits * sizeof(unsigned);
  s.pairs_bytes = s.passes > 1 ? Align256((size_t)s.m * sizeof(unsigned)) : 0;
  s.bytes = s.counts_bytes + s.groups_bytes + 2 * s.pairs_bytes;
  return s;
}

// ---------------------------------------------------------------- gradient
//
// The sorted pairs are cut into chunks of equal length, whatever the tokens are: a token that half of all bags name
// is the work of many waves.  A run of equal keys inside one chunk is summed and written there; of a run that goes on
// beyond its chunk each chunk leaves its part of the sum in the work memory, and a second launch (k_grad_join) adds
// the parts in order.

// First pair whose key is at least v: the whole wave asks, 64 probes a step (five steps for 2^30 pairs, where halving
// takes thirty loads one after the other).
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

  // Whether this workgroup writes zeros, and the how many-th of its kind it is.  The others start first: they wait for rows
  // that they gather, these only write (32,768 x 4096: 256 us, 272 the other way round, 445 in turns).
  __device__ __forceinline__ bool Fills(unsigned *block) const {
    const unsigned walk = gridDim.x - fill_blocks;
    const bool fills = blockIdx.x >= walk;
    *block = fills ? blockIdx.x - walk : blockIdx.x;
    return fills;
  }

  // kVec columns of row v from d on.  The first `skip` of them are another lane's, too: to be added only once.
  template <int kVec>
  __device__ __forceinline__ void Write(unsigned v, int d, int skip, const float (&sum)[kVec]) const {
    O *at = grad_table + (long long)v * table_stride + d;
    if (accumulate && skip > 0) {
      for (int c = 0; c < kVec; ++c)
        if (c >= skip) at[c] = Round<O>(static_cast<float>(at[c]) + sum[c] * scale);
      return;
    }
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
  __device__ __forceinline__ void Finish(unsigned v, unsigned w, int d, int skip, bool begins, bool ends, const float (&sum)[kVec]) const {
    if (v >= vocab) return;
    if (begins && ends) {
      Write<kVec>(v, d, skip, sum);
    } else {
      Pack<float, kVec> y;
#pragma unroll
      for (int c = 0; c < kVec; ++c) y.v[c] = sum[c];
      Store<float, kVec>(parts + ((size_t)w * 2 + (begins ? 1 : 0)) * dim + d, dim - d, y);
    }
  }
};

// Zeros for the rows [block * slots, ...) that no token names.  Which these are is found from the few pairs of those rows.
template <int kBlock, typename T, typename O>
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
  if (end - begin <= 8 * kBlock) {
    for (unsigned p = begin + threadIdx.x; p < end; p += kBlock) {
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
  // a row in pieces of 16 aligned bytes (past the caches: 345 -> 272 us where 0.8 GB are zeros; the sums are better
  // left in them, 267 and 274), elements at its ends
  constexpr int kVec = 16 / sizeof(O);
  const int pieces = g.dim / kVec + 2, lanes = min(64, pieces);
  const int groups = kBlock / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  if (group >= groups) return;
  for (unsigned k = group; k < slots; k += groups) {
    if (s_named[k / 32] >> (k % 32) & 1u) continue;
    O *row = g.grad_table + (long long)(v0 + k) * g.table_stride;
    const int before = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(O));  // elements of the first piece in front of the row
    for (int d = lane * kVec - before; d < g.dim; d += lanes * kVec) {
      if (d >= 0 && d + kVec <= g.dim) {
        typedef float Piece __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(Piece{0.0f, 0.0f, 0.0f, 0.0f}, reinterpret_cast<Piece *>(row + d));
      } else {
        for (int c = max(d, 0); c < min(d + kVec, g.dim); ++c) row[c] = O(0);
      }
    }
  }
}

// The runs of chunk w, columns [d, d + kVec): done(key, begins, ends, sum) for each, whether it begins and ends in
// the chunk. kAhead rows are in flight, and the pairs of the next step.
// kWave: the chunk is the whole wave's, and its keys and rows, which nobody writes meanwhile, are scalar loads.
template <bool kWave>
struct PairsAt {
  typedef const unsigned *Pointer;
};
template <>
struct PairsAt<true> {
  typedef const __attribute__((address_space(4))) unsigned *Pointer;
};
template <int kVec, bool kWave, typename T, typename O, typename Done>
__device__ __forceinline__ void WalkChunk(const Gradient<T, O> &g, unsigned w, int d, const Done &done) {
  typedef typename PairsAt<kWave>::Pointer Pointer;
  const Pointer keys = (Pointer)g.keys, rows = (Pointer)g.rows;
  const unsigned begin = w * g.chunk, end = min(g.m, begin + g.chunk);
  unsigned cur = keys[begin];
  bool begins = begin == 0 || keys[begin - 1] != cur;
  float sum[kVec];
#pragma unroll
  for (int c = 0; c < kVec; ++c) sum[c] = 0.0f;
  const T *from = g.grad_out + d;
  unsigned key[kAhead], row[kAhead], next_key[kAhead], next_row[kAhead];
  auto pairs = [&](unsigned p) {
    if (p + kAhead <= end) {
      typedef Pack<unsigned, kAhead> Some;
      if constexpr (kWave) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          next_key[k] = keys[p + k];
          next_row[k] = rows[p + k];
        }
      } else {
        *reinterpret_cast<Some *>(next_key) = *reinterpret_cast<const Some *>(keys + p);
        *reinterpret_cast<Some *>(next_row) = *reinterpret_cast<const Some *>(rows + p);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {  // past the end the last key stands, without a row
        const unsigned at = min(p + k, end - 1);
        next_key[k] = keys[at];
        next_row[k] = p + k < end ? rows[at] : g.n;
      }
    }
  };
  pairs(begin);
  for (unsigned p = begin; p < end; p += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      key[k] = next_key[k];
      row[k] = next_row[k];
    }
    // every load is asked for: what a pair has no row for is the last one's, and not added
    Pack<T, kVec> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      x[k] = *reinterpret_cast<const Pack<T, kVec> *>(from + (long long)min(row[k], g.n - 1u) * g.out_stride);
    if (p + kAhead < end) pairs(p + kAhead);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (key[k] != cur) {
        done(cur, begins, true, sum);
        cur = key[k];
        begins = true;
#pragma unroll
        for (int c = 0; c < kVec; ++c) sum[c] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < kVec; ++c) sum[c] += row[k] < g.n ? static_cast<float>(x[k].v[c]) : 0.0f;
    }
  }
  done(cur, begins, end == g.m || keys[end] != cur, sum);
}

// Rows of more than kNarrow elements: 2^lanes_log lanes hold kVec columns each and walk a chunk pair by pair.
template <typename T, typename O, int kVec, bool kWave>
__global__ void __launch_bounds__(kThreads) k_grad_wide(const Gradient<T, O> g) {
  unsigned block;
  if (g.Fills(&block)) {
    FillRows<kThreads>(g, block);
    return;
  }
  const unsigned piece = block % g.pieces;
  const int lanes_log = kWave ? 6 : g.lanes_log;
  unsigned w = ((block / g.pieces) * kThreads + threadIdx.x) >> lanes_log;
  if constexpr (kWave) w = __builtin_amdgcn_readfirstlane(w);
  const int column = (int)(((piece << lanes_log) + (threadIdx.x & ((1u << lanes_log) - 1u))) * kVec);
  if (w >= g.chunks || column >= g.dim) return;
  const int d = min(column, g.dim - kVec);
  WalkChunk<kVec, kWave>(g, w, d, [&](unsigned v, bool begins, bool ends, const float (&sum)[kVec]) {
    g.template Finish<kVec>(v, w, d, column - d, begins, ends, sum);
  });
}

// The same for so few pairs that one workgroup holds all chunks of a piece: the parts of runs that go on meet in the
// LDS, and there is no second launch (64 pairs x 64: 5.8 us; with it 6.2 and 2.2, and 3.5 more of the host).
constexpr int kFewThreads = 1024;
constexpr unsigned kFewPairs = 512;
constexpr long long kMostFewRows = 1ll << 29;
template <typename T, typename O, int kVec>
__global__ void __launch_bounds__(kFewThreads) k_grad_few(const Gradient<T, O> g) {
  unsigned block;
  if (g.Fills(&block)) {
    FillRows<kFewThreads>(g, block);
    return;
  }
  __shared__ float s_part[kVec][kFewThreads];  // of the run that comes in
  const unsigned w = threadIdx.x >> g.lanes_log;
  const int column = (int)(((block << g.lanes_log) + (threadIdx.x & ((1u << g.lanes_log) - 1u))) * kVec);
  const int d = min(column, g.dim - kVec);
  const bool live = w < g.chunks && column < g.dim;
  unsigned goes_on = g.vocab;  // key of the run that goes on
  float rest[kVec];
#pragma unroll
  for (int c = 0; c < kVec; ++c) rest[c] = 0.0f;
  if (live) {
    WalkChunk<kVec, false>(g, w, d, [&](unsigned v, bool begins, bool ends, const float (&sum)[kVec]) {
      if (v >= g.vocab) return;
      if (begins && ends) {
        g.template Write<kVec>(v, d, column - d, sum);
      } else if (begins) {
        goes_on = v;
#pragma unroll
        for (int c = 0; c < kVec; ++c) rest[c] = sum[c];
      } else {
#pragma unroll
        for (int c = 0; c < kVec; ++c) s_part[c][threadIdx.x] = sum[c];
      }
    });
  }
  __syncthreads();
  if (goes_on >= g.vocab) return;
  for (unsigned x = w + 1; x < g.chunks && g.keys[x * g.chunk] == goes_on; ++x) {
#pragma unroll
    for (int c = 0; c < kVec; ++c) rest[c] += s_part[c][threadIdx.x + ((x - w) << g.lanes_log)];
  }
  g.template Write<kVec>(goes_on, d, column - d, rest);
}

__device__ __forceinline__ float WaveSum(float v) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Rows of up to kDim <= kNarrow elements: a lane takes a pair with its whole row, a wave 64 pairs of a chunk at a
// time.  While the key stays the same the lanes add up what is theirs; when it changes they meet.
template <typename T, typename O, int kDim>
__global__ void __launch_bounds__(kThreads) k_grad_narrow(const Gradient<T, O> g) {
  unsigned block;
  if (g.Fills(&block)) {
    FillRows<kThreads>(g, block);
    return;
  }
  const unsigned w = __builtin_amdgcn_readfirstlane((block * kThreads + threadIdx.x) >> 6);
  if (w >= g.chunks) return;
  const unsigned lane = threadIdx.x & 63u;
  const unsigned begin = w * g.chunk, end = min(g.m, begin + g.chunk);
  unsigned cur = g.keys[begin];
  bool begins = begin == 0 || g.keys[begin - 1] != cur;
  float sum[kDim];
#pragma unroll
  for (int c = 0; c < kDim; ++c) sum[c] = 0.0f;
  constexpr int kRounds = kDim == 1 ? 8 : 4;
  for (unsigned p = begin; p < end; p += 64 * kRounds) {
    unsigned key[kRounds], row[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {  // past the end the last key stands, without a row
      const unsigned at = p + k * 64 + lane;
      key[k] = __builtin_nontemporal_load(g.keys + min(at, end - 1));
      row[k] = __builtin_nontemporal_load(g.rows + min(at, end - 1));
      if (at >= end) row[k] = g.n;
    }
    float x[kRounds][kDim];
    if (g.dim == kDim) {
      Pack<T, kDim> held[kRounds];
#pragma unroll
      for (int k = 0; k < kRounds; ++k)
        held[k] = *reinterpret_cast<const Pack<T, kDim> *>(g.grad_out + (long long)min(row[k], g.n - 1u) * g.out_stride);
#pragma unroll
      for (int k = 0; k < kRounds; ++k)
#pragma unroll
        for (int c = 0; c < kDim; ++c) x[k][c] = static_cast<float>(held[k].v[c]);
    } else {
#pragma unroll
      for (int k = 0; k < kRounds; ++k)
#pragma unroll
        for (int c = 0; c < kDim; ++c)
          x[k][c] = static_cast<float>(g.grad_out[(long long)min(row[k], g.n - 1u) * g.out_stride + min(c, g.dim - 1)]);
    }
#pragma unroll
    for (int k = 0; k < kRounds; ++k)
#pragma unroll
      for (int c = 0; c < kDim; ++c) x[k][c] = row[k] < g.n ? x[k][c] : 0.0f;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const bool same = key[k] == cur;
      if (__ballot(!same) == 0ull) {
#pragma unroll
        for (int c = 0; c < kDim; ++c) sum[c] += x[k][c];
        continue;
      }
      // the run that came in ends here
      float total[kDim];
#pragma unroll
      for (int c = 0; c < kDim; ++c) total[c] = WaveSum(sum[c] + (same ? x[k][c] : 0.0f));
      if (lane == 0) g.template Finish<kDim>(cur, w, 0, 0, begins, true, total);
      // the last key goes on; those between are whole: sums over runs of equal keys, by steps of doubled length
      const unsigned last = __builtin_amdgcn_readlane(key[k], 63);
      const bool between = !same && key[k] != last;
      if (__ballot(between) != 0ull) {
        float run[kDim];
#pragma unroll
        for (int c = 0; c < kDim; ++c) run[c] = x[k][c];
        for (int off = 1; off < 64; off <<= 1) {
          const bool joins = __shfl_up(key[k], off) == key[k] && lane >= (unsigned)off;
#pragma unroll
          for (int c = 0; c < kDim; ++c) {
            const float o = __shfl_up(run[c], off);
            if (joins) run[c] += o;
          }
        }
        const unsigned after = __shfl_down(key[k], 1);
        if (between && after != key[k]) g.template Finish<kDim>(key[k], w, 0, 0, true, true, run);
      }
#pragma unroll
      for (int c = 0; c < kDim; ++c) sum[c] = key[k] == last ? x[k][c] : 0.0f;
      cur = last;
      begins = true;
    }
  }
  float total[kDim];
#pragma unroll
  for (int c = 0; c < kDim; ++c) total[c] = WaveSum(sum[c]);
  if (lane == 0) g.template Finish<kDim>(cur, w, 0, 0, begins, end == g.m || g.keys[end] != cur, total);
}

// Chunk w: whether a run begins in it that goes on beyond its end, and the last chunk that run reaches.
template <typename T, typename O>
__device__ __forceinline__ bool GoesOn(const Gradient<T, O> &g, unsigned w, unsigned *v, unsigned *last) {
  const unsigned begin = w * g.chunk, end = begin + g.chunk;
  if (w >= g.chunks || end >= g.m) return false;
  const unsigned next = g.keys[end], same = g.keys[end - 1], first = g.keys[begin], before = g.keys[max(begin, 1u) - 1u];
  *v = next;
  if (next >= g.vocab || same != next || (begin != 0 && first == next && before == next)) return false;
  // the chunks after it that the run still begins: most often one or two, so 64 are asked at once
  const unsigned x = w + 1u + (threadIdx.x & 63u);
  const unsigned long long other = ~__ballot(x < g.chunks && g.keys[(size_t)min(x, g.chunks - 1u) * g.chunk] == next);
  if (other != 0ull) *last = w + (unsigned)__builtin_ctzll(other);
  else *last = (WaveLowerBound(g.keys + end, g.m - end, next + 1u) + end - 1u) / g.chunk;
  return true;
}

// The parts of the runs that go on, added up: every wave asks for a chunk of its own and sums the run that begins
// there, 2^lanes_log lanes side by side over the columns (four each) and the others over the parts.  A run of many
// parts is left to all waves of the workgroup.
constexpr int kJoinVec = 4;
constexpr unsigned kManyParts = 8;  // of a lane
template <int kJoinThreads, typename T, typename O>
__global__ void __launch_bounds__(kJoinThreads) k_grad_join(const Gradient<T, O> g, int lanes_log) {
  constexpr unsigned kWaves = kJoinThreads / 64;
  __shared__ float s_sum[kWaves][64][kJoinVec];
  __shared__ unsigned s_key[kWaves], s_last[kWaves];
  const unsigned lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned share = lane >> lanes_log, shares = 64u >> lanes_log;  // of the parts, within the wave
  const int column = (int)(lane & ((1u << lanes_log) - 1u)) * kJoinVec, step = kJoinVec << lanes_log;
  float sum[kJoinVec];
  // parts of the run from chunk w on, beginning with the `from`-th and taking every `by`-th: the first is what the
  // run left in w itself
  auto add = [&](unsigned w, unsigned last, int d, unsigned from, unsigned by) {
#pragma unroll
    for (int c = 0; c < kJoinVec; ++c) sum[c] = 0.0f;
    if (d >= g.dim) return;
#pragma unroll 8
    for (unsigned x = w + from; x <= last; x += by) {
      Pack<float, kJoinVec> y;
      Load<float, kJoinVec>(g.parts + ((size_t)x * 2 + (x == w ? 1 : 0)) * g.dim + d, g.dim - d, &y);
#pragma unroll
      for (int c = 0; c < kJoinVec; ++c) sum[c] += y.v[c];
    }
  };
  auto meet = [&] {
    for (int off = 32; off >= 1 << lanes_log; off >>= 1)
#pragma unroll
      for (int c = 0; c < kJoinVec; ++c) sum[c] += __shfl_xor(sum[c], off);
  };
  const unsigned w0 = blockIdx.x * kWaves;
  unsigned v = 0, last = 0;
  const bool goes = GoesOn(g, w0 + wave, &v, &last), many = goes && last - (w0 + wave) > kManyParts * shares;
  if (goes && !many) {
    for (int d0 = (int)blockIdx.y * step; d0 < g.dim; d0 += (int)gridDim.y * step) {
      add(w0 + wave, last, d0 + column, share, shares);
      meet();
      if (share == 0 && d0 + column < g.dim) g.template Write<kJoinVec>(v, d0 + column, 0, sum);
    }
  }
  if (lane == 0) {
    s_key[wave] = v;
    s_last[wave] = many ? last : 0u;  // (a run that goes on ends behind chunk 0)
  }
  __syncthreads();
  for (unsigned k = 0; k < kWaves; ++k) {
    if (s_last[k] == 0u) continue;
    for (int d0 = (int)blockIdx.y * step; d0 < g.dim; d0 += (int)gridDim.y * step) {
      add(w0 + k, s_last[k], d0 + column, wave * shares + share, kWaves * shares);
      meet();
#pragma unroll
      for (int c = 0; c < kJoinVec; ++c) s_sum[wave][lane][c] = sum[c];
      __syncthreads();
      if (wave == 0 && share == 0 && d0 + column < g.dim) {
        for (unsigned x = 1; x < kWaves; ++x)
#pragma unroll
          for (int c = 0; c < kJoinVec; ++c) sum[c] += s_sum[x][lane][c];
        g.template Write<kJoinVec>(s_key[k], d0 + column, 0, sum);
      }
      __syncthreads();
    }
  }
}

// Pairs of a chunk: few, so that there are waves for every CU, and more where there are enough (4096), since each
// chunk leaves two rows of parts to be joined; and so few that a launch counts its threads with 32 bits.  Waves are
// counted as if every lane held eight elements and none were idle: four million by this count are at most sixteen
// (rows of 257 to 264 elements of 32 bits), 2^30 threads beside the 2^31 that zeros take.  (5,003 x 771: 28 us with
// 16 pairs, 42 with 64; 64 x 64: 7 and 17; 32,768 x 4096, parts and all: 385 us with 16, 366 with 64.)
unsigned ChunkOf(unsigned m, int dim) {
  const bool wide = dim > kNarrow;
  const unsigned most = wide ? 256 : 1024;
  const unsigned long long per_64 = wide ? (dim + 7) / 8 : 64;  // waves of 64 chunks
  unsigned c = wide ? 16 : m <= most ? most : 64;  // (few narrow pairs: one wave, and nothing to join)
  while ((c < most && m / c * per_64 / 64 > (wide ? 4096 : 16384)) || m / c * per_64 / 64 > (1 << 22)) c *= 2;
  return c;
}

// ------------------------------------------------------------------ checks

constexpr int kMostDim = 65535 * 256;  // (a grid's second dimension counts 65,535 pieces of a row of 256 elements at least)

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
  if (plan.ranges > 0) {
    WithToken(a.bags.bits, [&](auto token) {
      typedef decltype(token) Token;
      const Pairs<Token> in = PairsOf<Token>(a.bags, plan.m);
      auto launch = [&](auto rounds) {
        hipLaunchKernelGGL((k_sort_ranges<decltype(rounds)::value, Token>), dim3(plan.ranges), dim3(kRangeThreads), 0, st, in, plan.span,
                           plan.key_bits, plan.place_bits, a.keys, a.rows);
      };
      if (plan.m <= 1 * kRangeThreads) launch(std::integral_constant<int, 1>());
      else if (plan.m <= 4 * kRangeThreads) launch(std::integral_constant<int, 4>());
      else if (plan.m <= 8 * kRangeThreads) launch(std::integral_constant<int, 8>());
      else if (plan.m <= 16 * kRangeThreads) launch(std::integral_constant<int, 16>());
      else launch(std::integral_constant<int, 32>());
    });
    HIP_OK(hipGetLastError());
    return;
  }
  unsigned char *work = static_cast<unsigned char *>(a.work);
  unsigned *counts = reinterpret_cast<unsigned *>(work);
  unsigned *groups = reinterpret_cast<unsigned *>(work + plan.counts_bytes);
  unsigned *spare[2];
  spare[0] = groups + plan.groups_bytes / sizeof(unsigned);
  spare[1] = spare[0] + plan.pairs_bytes / sizeof(unsigned);
  unsigned *last[2] = {a.keys, a.rows};
  for (int pass = 0; pass < plan.passes; ++pass) {
    // the last pass writes to the caller's arrays, the passes before it in turn
    unsigned **to = (plan.passes - 1 - pass) % 2 == 0 ? last : spare, **from = to == last ? spare : last;
    const Digit digit{pass * plan.bits, plan.bits, (1u << plan.bits) - 1u};
    auto launch = [&](const auto &in) {
      typedef std::decay_t<decltype(in)> Source;
      auto few = [&](auto pairs) {
        constexpr int kPairs = decltype(pairs)::value;
        hipLaunchKernelGGL((k_sort_count<kPairs, Source>), dim3(plan.tiles), dim3(kSortThreads), 0, st, in, digit, counts);
        hipLaunchKernelGGL((k_sort_scatter<kPairs, true, Source>), dim3(plan.tiles), dim3(kSortThreads), 0, st, in, digit, plan.tiles,
                           counts, nullptr, nullptr, to[0], to[1]);
      };
      if (plan.groups > 1) {
        hipLaunchKernelGGL((k_sort_count<kSortRounds, Source>), dim3(plan.tiles), dim3(kSortThreads), 0, st, in, digit, counts);
        hipLaunchKernelGGL(k_sort_sum_tiles, dim3(plan.groups), dim3(kDigits), 0, st, counts, plan.tiles, groups);
        hipLaunchKernelGGL(k_sort_sum_groups, dim3(kDigits / 64), dim3(1024), 0, st, groups, plan.groups);
        hipLaunchKernelGGL((k_sort_scatter<kSortRounds, false, Source>), dim3((plan.tiles + kXcds - 1) / kXcds * kXcds),
                           dim3(kSortThreads), 0, st, in, digit, plan.tiles, counts, groups, groups + (size_t)plan.groups * kDigits, to[0],
                           to[1]);
      } else if (plan.pairs == 2) {
        few(std::integral_constant<int, 2>());
      } else if (plan.pairs == 4) {
        few(std::integral_constant<int, 4>());
      } else {
        few(std::integral_constant<int, 8>());
      }
    };
    if (pass > 0) {
      launch(FromPairs{from[0], from[1], plan.m});
    } else {
      WithToken(a.bags.bits, [&](auto token) {
        typedef decltype(token) Token;
        launch(FromTokens<Token>{PairsOf<Token>(a.bags, plan.m), plan.m});
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
  if (a.table_type != kFloat32 && a.table_type != a.type)
    throw std::runtime_error("the table's gradient is float32 or of the type of grad_out");
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
    // rows of zeros a workgroup: 16 KB of them for every four waves (more where a launch would count its threads
    // beyond 32 bits)
    auto fill = [&](int threads) {
      g.slots = (unsigned)std::min<size_t>(std::max<size_t>(64 * threads / (a.dim * sizeof(O)), 1), kMostSlots);
      while (g.slots < kMostSlots && a.vocab / g.slots > (1 << 22) / (threads / kThreads)) g.slots *= 2;
      g.slots = std::min(g.slots, kMostSlots);
      g.fill_blocks = a.accumulate ? 0 : (unsigned)((a.vocab + g.slots - 1) / g.slots);
    };
    fill(kThreads);
    g.lanes_log = 6;
    g.pieces = 1;
    if (a.dim > kNarrow) {
      constexpr int kVec = 16 / sizeof(T);
      const unsigned vectors = (unsigned)(a.dim + kVec - 1) / kVec;
      g.lanes_log = std::min(LogAtLeast(vectors), 6);
      g.pieces = (vectors + (1u << g.lanes_log) - 1) >> g.lanes_log;
      const unsigned walkers = kFewThreads >> g.lanes_log;
      // (256 rows a workgroup and 1024 threads: a launch counts threads with 32 bits)
      const bool counts = a.accumulate || a.vocab <= kMostFewRows;
      if (m > 0 && m <= std::min(kFewPairs, 32 * walkers) && counts) {
        fill(kFewThreads);
        g.chunk = (m + walkers - 1) / walkers;
        g.chunks = (m + g.chunk - 1) / g.chunk;
        hipLaunchKernelGGL((k_grad_few<T, O, kVec>), dim3(g.pieces + g.fill_blocks), dim3(kFewThreads), 0, st, g);
        return;
      }
      const unsigned long long blocks =
          ((((unsigned long long)g.chunks << g.lanes_log) + kThreads - 1) / kThreads) * g.pieces + g.fill_blocks;
      const dim3 grid((unsigned)blocks), block(kThreads);
      if (blocks > 0 && g.lanes_log == 6) hipLaunchKernelGGL((k_grad_wide<T, O, kVec, true>), grid, block, 0, st, g);
      else if (blocks > 0) hipLaunchKernelGGL((k_grad_wide<T, O, kVec, false>), grid, block, 0, st, g);
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
    }
    if (g.chunks > 1) {
      const int lanes_log = std::min(LogAtLeast((a.dim + kJoinVec - 1) / kJoinVec), 6);
      const int pieces = (a.dim + 64 * kJoinVec - 1) / (64 * kJoinVec);
      auto join = [&](auto threads) {
        constexpr unsigned kJoin = decltype(threads)::value, kWaves = kJoin / 64;
        hipLaunchKernelGGL((k_grad_join<kJoin, T, O>), dim3((g.chunks + kWaves - 1) / kWaves, std::min(pieces, 16)), dim3(kJoin), 0, st, g,
                           lanes_log);
      };
      // few chunks: the longest run is what takes time, and eight waves share it (100,000 pairs x 256, one token in
      // sixteen the same: 22 us, 37 by four); many: the workgroups that find nothing to do (50 M narrow pairs: 27 us
      // by four, 32 by eight)
      if (g.chunks < 32768) join(std::integral_constant<int, 512>());
      else join(std::integral_constant<int, 256>());
    }
  };
  WithType(a.type, [&](auto t) {
    if (a.table_type == kFloat32) launch(t, float());
    else launch(t, t);
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
