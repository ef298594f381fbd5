// Log probabilities of given tokens under rows of logits, the entropy of each row, its likeliest tokens, and the gradient
// of the logits.  With a_j = scale (x_j - max x) and S = sum exp a_j,
//   log_prob = a_token - log S,   entropy = log S - (sum a_j exp a_j) / S,
//   grad_j   = scale (g ([j = token] - p_j) - h p_j (log p_j + entropy)),   p_j = exp(a_j - log S).
// A row is read once: maximum, S and sum a exp a run along it, and a new maximum scales what was summed before
// (sum (a + d) exp (a + d) = exp d (sum a exp a + d sum exp a)).  The gradient reads the row once more: what must be known of all of it, the maximum and
// log S, is kept in 8 bytes a row.  Reading and writing the logits bounds both (4096 x 131,072 bf16: 1 GiB read in 212 us, read and written in 362, 5.1 and 5.9
// TB/s); with the likeliest tokens the search for them, where rows are short.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "operators_device.h"

namespace arb {
namespace {

typedef unsigned long long Key;  // value (in an order of whole numbers) and inverted index: the greater one comes first; 0: none

constexpr int kMostTop = 64;     // of them a wave holds one a lane
constexpr int kMostParts = 32;   // of a row, joined by a wave
constexpr long long kPart = 8192;  // a row is not cut into less: 16 KB, a workgroup's loads in one go
constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -1000.0f;  // exponents (of two) below are taken for it where they are factors: their power is 0, and must not meet an infinity

__device__ __forceinline__ float Infinity() { return __builtin_inff(); }
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ unsigned OrderOf(float value) {
  const unsigned bits = __float_as_uint(value + 0.0f);  // (-0 and 0 are equal)
  return bits ^ ((bits >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ Key KeyOf(float value, unsigned index) { return ((Key)OrderOf(value) << 32) | (Key)(~index); }
__device__ __forceinline__ float ValueOf(Key key) {
  const unsigned order = (unsigned)(key >> 32);
  return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ unsigned IndexOf(Key key) { return ~(unsigned)key; }

__device__ __forceinline__ Key LaneKey(Key key, int lane) {
  const unsigned low = __builtin_amdgcn_readlane((int)(unsigned)key, lane), high = __builtin_amdgcn_readlane((int)(unsigned)(key >> 32), lane);
  return ((Key)high << 32) | low;
}

// The greatest word that at least `k` of a wave's words (kEach a lane) are no less than, bit by bit from the top; or, as soon as
// some word has exactly k on its side, that one.
template <int kEach, typename Word>
__device__ __forceinline__ Word Least(const Word (&words)[kEach], int k) {
  Word least = 0;
  for (int bit = sizeof(Word) * 8 - 1; bit >= 0; --bit) {
    const Word tried = least | (Word)1 << bit;
    int count = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) count += __popcll(__ballot(words[e] >= tried));
    if (count >= k) least = tried;
    if (count == k) break;
  }
  return least;
}

// A wave's list of 64 keys in order, one a lane: `one` takes its place, and the last one falls out.
__device__ __forceinline__ void Insert(Key *held, Key one) {
  const int lane = threadIdx.x & 63, place = __popcll(__ballot(*held > one));
  const auto lane_before = [](unsigned word) { return (unsigned)__builtin_amdgcn_update_dpp((int)word, (int)word, 0x138, 0xF, 0xF, false); };
  const Key before = ((Key)lane_before((unsigned)(*held >> 32)) << 32) | lane_before((unsigned)*held);
  *held = lane < place ? *held : lane == place ? one : before;
}

// Sums of (a part of) a row: the maximum, sum 2^d and sum d 2^d of d = log2(e) scale (x - maximum).
struct Sums {
  float most, sum, moment;
};

// `most` where nothing but minus infinity was seen is no base to subtract.
__device__ __forceinline__ float Base(float most) { return most == -Infinity() ? 0.0f : most; }

__device__ __forceinline__ Sums Join(const Sums &a, const Sums &b, float factor) {
  const float most = fmaxf(a.most, b.most), base = Base(most);
  const float da = factor * (a.most - base), db = factor * (b.most - base);  // (minus infinity where one has nothing)
  const float ea = Exp2(da), eb = Exp2(db);
  Sums r;
  r.most = most;
  r.sum = ea * a.sum + eb * b.sum;
  r.moment = ea * (a.moment + fmaxf(da, kLowest) * a.sum) + eb * (b.moment + fmaxf(db, kLowest) * b.sum);
  return r;
}

// All lanes' values by op, whose order does not matter to it but for rounding (which is the same in every lane): neighbours, pairs, then mirrored halves of 16
// lanes by instructions that take an operand from another lane, then the halves of 32 and of all.  (__shfl_xor goes through the LDS each time.)
template <typename Op>
__device__ __forceinline__ float OfLanes(float v, const Op &op) {
  const auto other = [](float x, auto how) {
    const int w = __float_as_int(x);
    return __int_as_float(__builtin_amdgcn_update_dpp(w, w, decltype(how)::value, 0xF, 0xF, false));
  };
  v = op(v, other(v, std::integral_constant<int, 0xB1>()));   // lanes 1 0 3 2 of four
  v = op(v, other(v, std::integral_constant<int, 0x4E>()));   // lanes 2 3 0 1
  v = op(v, other(v, std::integral_constant<int, 0x141>()));  // eight mirrored
  v = op(v, other(v, std::integral_constant<int, 0x140>()));  // sixteen mirrored
  const auto sixteens = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(sixteens[0]), __uint_as_float(sixteens[1]));
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
}

// The lanes' sums joined: their maximum first, to which each takes its own.
template <bool kMoment>
__device__ __forceinline__ Sums JoinLanes(const Sums &s, float factor) {
  Sums r;
  r.most = OfLanes(s.most, [](float a, float b) { return fmaxf(a, b); });
  const float d = factor * (s.most - Base(r.most)), e = Exp2(d);
  const auto add = [](float a, float b) { return a + b; };
  r.sum = OfLanes(e * s.sum, add);
  r.moment = kMoment ? OfLanes(e * (s.moment + fmaxf(d, kLowest) * s.sum), add) : 0.0f;
  return r;
}

struct RowsArgs {
  const void *logits;
  long long row_stride, class_stride;
  long long n;
  unsigned vocab;
  float scale, factor;  // factor: scale * log2(e)
  const void *tokens;
  int token_bits;
  float *log_probs, *entropy;
  float2 *stats;
  int top;
  int *top_tokens;
  float *top_log_probs;
  unsigned *status;
  // rows in parts
  int parts;
  unsigned part;  // classes of each
  float4 *sums;   // [n][parts]
  Key *keys;      // [n][parts][top]
};

__device__ __forceinline__ long long TokenAt(const RowsArgs &a, long long i) {
  return a.token_bits == 32 ? (long long)static_cast<const int *>(a.tokens)[i] : static_cast<const long long *>(a.tokens)[i];
}

// log S; 0 for a row that has nothing but minus infinity (whose maximum tells it).  A NaN or plus infinity makes it a NaN.
__device__ __forceinline__ float LogSum(const Sums &s) { return s.sum == 0.0f ? 0.0f : logf(s.sum); }

// What a row answers with, but for its top.
template <typename T>
__device__ __forceinline__ void WriteRow(const RowsArgs &a, const Sums &s, float log_sum, long long i) {
  if (a.log_probs != nullptr) {
    const long long t = TokenAt(a, i);
    float v = 0.0f;
    if (t >= 0 && t < (long long)a.vocab) {
      const float x = (float)static_cast<const T *>(a.logits)[i * a.row_stride + t * a.class_stride];
      v = a.scale * (x - Base(s.most)) - log_sum;
    } else if (t != -1 && a.status != nullptr) {
      *a.status = 1u;
    }
    a.log_probs[i] = v;
  }
  if (a.entropy != nullptr) {
    // (ln 2 takes the moment back to exponents of e)
    const float h = s.sum == 0.0f ? 0.0f : log_sum - kLn2 * (s.moment / s.sum);
    a.entropy[i] = h;
  }
  if (a.stats != nullptr) a.stats[i] = make_float2(s.most, log_sum);
}

__device__ __forceinline__ void WriteTop(const RowsArgs &a, const Sums &s, float log_sum, long long i, int rank, float value, unsigned index) {
  const bool none = log_sum != log_sum;  // a row with a NaN, or plus infinity
  a.top_tokens[i * a.top + rank] = none ? -1 : (int)index;
  a.top_log_probs[i * a.top + rank] = a.scale * (value - Base(s.most)) - log_sum;
}
__device__ __forceinline__ void WriteTop(const RowsArgs &a, const Sums &s, float log_sum, long long i, int rank, Key key) {
  WriteTop(a, s, log_sum, i, rank, ValueOf(key), IndexOf(key));
}

// ------------------------------------------------------------------ a row a team

// A team of kWaves waves reads a row, or a part of one; one wave a row: four teams a workgroup.  kSide: classes side by side, read 16 bytes a lane (777 x 50,021
// fp16 20.4 us, 3.8 TB/s; rows of an odd length begin anywhere, and loads at less than four bytes' alignment take longer: 8192 x 50,021 bf16 171 us, x 50,024 145;
// vectors from where 16 bytes begin would make a row's last bits depend on where it lies).
// The likeliest tokens: every thread keeps the maximum of what it reads.  The k-th greatest of these maxima has k elements of the row on
// its side, so the k likeliest are no less than it, and whatever is no less lies with the threads whose maxima are no less: about k
// of 256, so that only their share of the row is read again.  (Where many are equal, as in a row of one value, more is.)  777 x 50,021 fp16 top 5: 26.7 us, 6
// of them for this.
template <typename T, int kWaves, int kUnroll, bool kSide, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kWaves == 1 ? 256 : kWaves * 64) k_rows(const RowsArgs a) {
  constexpr int kVec = 16 / sizeof(T), kTeam = kWaves * 64, kTeams = kWaves == 1 ? 4 : 1, kChunk = kUnroll * kVec;
  __shared__ Sums s_sums[kWaves];
  __shared__ unsigned s_most[kTop ? kTeams : 1][kTop ? kTeam : 1];
  __shared__ unsigned short s_owners[kTop ? kTeams * kWaves : 1][kTop ? 64 : 1];
  __shared__ Key s_lists[kTop && kWaves > 1 ? kWaves : 1][kTop && kWaves > 1 ? kMostTop : 1];
  const int lane = threadIdx.x & 63, wave = kWaves == 1 ? 0 : threadIdx.x >> 6, team = kWaves == 1 ? threadIdx.x >> 6 : 0;
  const unsigned t = kWaves == 1 ? lane : threadIdx.x;
  const long long items = a.n * a.parts;
  // (all teams of a workgroup go the same number of rounds: there are barriers inside)
  for (long long first = (long long)blockIdx.x * kTeams; first < items; first += (long long)gridDim.x * kTeams) {
    const long long item = first + team;
    const bool live = item < items;
    const long long row = live ? item / a.parts : 0;
    const unsigned part = live ? (unsigned)(item - row * a.parts) : 0;
    const unsigned begin = part * a.part, length = live ? min(a.part, a.vocab - begin) : 0;
    const long long apart = kSide ? 1 : a.class_stride;
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride + begin * apart;
    const auto vector_at = [&](unsigned at) {
      if constexpr (kSide) {
        return *reinterpret_cast<const Pack<T, kVec> *>(x + at);
      } else {
        Pack<T, kVec> p;
#pragma unroll
        for (int c = 0; c < kVec; ++c) p.v[c] = x[(at + c) * apart];
        return p;
      }
    };

    Sums s = {-Infinity(), 0.0f, 0.0f};
    const auto add = [&](const float (&v)[kChunk]) {
      float most = v[0];
#pragma unroll
      for (int c = 1; c < kChunk; ++c) most = fmaxf(most, v[c]);
      if (most > s.most) {
        const float d = a.factor * (s.most - most), e = Exp2(d);
        if (kEntropy) s.moment = e * (s.moment + fmaxf(d, kLowest) * s.sum);
        s.sum *= e;
        s.most = most;
      }
      const float base = Base(s.most);
#pragma unroll
      for (int c = 0; c < kChunk; ++c) {
        const float d = a.factor * (v[c] - base), e = Exp2(d);
        s.sum += e;
        if (kEntropy) s.moment = fmaf(fmaxf(d, kLowest), e, s.moment);
      }
    };
    const unsigned vectors = (length + kVec - 1) / kVec, whole = length / (kTeam * kChunk) * kUnroll;
    for (unsigned i = 0; i < whole; i += kUnroll) {
      Pack<T, kVec> p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = vector_at(((i + u) * kTeam + t) * kVec);
      float v[kChunk];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int c = 0; c < kVec; ++c) v[u * kVec + c] = (float)p[u].v[c];
      add(v);
    }
    if ((size_t)whole * kTeam + t < vectors) {  // the rest; what is beyond the end counts as minus infinity
      float v[kChunk];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const unsigned at = ((whole + u) * kTeam + t) * kVec;
        const bool all = at < length && length - at >= kVec;
        Pack<T, kVec> p;
        if (all) p = vector_at(at);
#pragma unroll
        for (int c = 0; c < kVec; ++c) v[u * kVec + c] = all ? (float)p.v[c] : at < length && c < (int)(length - at) ? (float)x[(at + c) * apart] : -Infinity();
      }
      add(v);
    }
    const unsigned mine = kTop && t < vectors ? OrderOf(s.most) : 0;

    // the sums of the team
    s = JoinLanes<kEntropy>(s, a.factor);
    if (kWaves > 1) {
      if (lane == 0) s_sums[wave] = s;
      __syncthreads();
      s = s_sums[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) s = Join(s, s_sums[w], a.factor);
    }
    const float log_sum = LogSum(s);
    if (live && t == 0) {
      if (a.parts == 1) WriteRow<T>(a, s, log_sum, row);
      else a.sums[item] = make_float4(s.most, s.sum, s.moment, 0.0f);
    }

    if constexpr (kTop) {
      unsigned words[kWaves];
      if constexpr (kWaves > 1) {
        s_most[0][t] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) words[w] = s_most[0][w * 64 + lane];
      } else {
        words[0] = mine;
      }
      const unsigned least = Least<kWaves>(words, a.top);
      // the wave's own threads of those, and their vectors, shared out over its lanes
      const unsigned long long owners = __ballot(mine != 0 && mine >= least);
      unsigned short *list = s_owners[team * kWaves + wave];
      if (owners >> lane & 1) list[__popcll(owners & ((1ull << lane) - 1))] = (unsigned short)t;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
      __builtin_amdgcn_wave_barrier();
      const unsigned rounds = (vectors + kTeam - 1) / kTeam, count = (unsigned)__popcll(owners) * rounds;
      Key held = 0;
      for (unsigned e0 = 0; e0 < count; e0 += 64) {
        const unsigned e = min(e0 + lane, count - 1), owner = e / rounds, at = ((e - owner * rounds) * kTeam + list[owner]) * kVec;
        const unsigned there = e0 + lane < count && at < length ? min(length - at, (unsigned)kVec) : 0;
        Pack<T, kVec> p;
        if (there == kVec) {
          p = vector_at(at);
        } else {
#pragma unroll
          for (int c = 0; c < kVec; ++c) p.v[c] = (unsigned)c < there ? x[(at + c) * apart] : T(0);
        }
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
          const Key key = (unsigned)c < there ? KeyOf((float)p.v[c], begin + at + c) : 0;
          const Key last = LaneKey(held, a.top - 1);
          unsigned long long found = __ballot((unsigned)(key >> 32) >= least && key > last);
          while (found != 0) {
            Insert(&held, LaneKey(key, __builtin_ctzll(found)));
            found &= found - 1;
          }
        }
      }
      // the wave's list meets the others': a key's place is how many are greater, in each of them
      int place = lane;
      if constexpr (kWaves > 1) {
        s_lists[wave][lane] = held;
        __syncthreads();
        int greater[kWaves] = {};
#pragma unroll
        for (int step = 64; step > 0; step /= 2) {  // (halving, in all lists at once; the last step twice: there may be 64)
          const int by = max(step / 2, 1);
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            if (greater[w] + by <= kMostTop && s_lists[w][greater[w] + by - 1] > held) greater[w] += by;
        }
#pragma unroll
        for (int w = 0; w < kWaves; ++w) place += w == wave ? 0 : greater[w];
      }
      // (with a NaN in it nothing is in order; a part shorter than the list leaves places empty)
      const bool broken = log_sum != log_sum;
      if (live && !broken && held != 0 && lane < a.top && place < a.top) {
        if (a.parts == 1) WriteTop(a, s, log_sum, row, place, held);
        else a.keys[item * a.top + place] = held;
      }
      if (live && wave == 0 && lane < a.top && (broken || (unsigned)lane >= length)) {
        if (a.parts == 1) WriteTop(a, s, log_sum, row, lane, 0);
        else a.keys[item * a.top + lane] = 0;
      }
    }
    if (kWaves > 1) __syncthreads();
  }
}

// The parts of a row, by one wave: a lane holds a part's sums and kEach of the parts' keys.  (5 us for 16 parts of 20 keys: a launch and one chain of loads, sums
// and choices, whatever the row.)
template <typename T, int kEach>
__global__ void __launch_bounds__(64) k_join(const RowsArgs a) {
  __shared__ Key s_top[kMostTop];
  const int lane = threadIdx.x;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    Sums s = {-Infinity(), 0.0f, 0.0f};
    Key words[kEach];
    const Key *keys = a.keys + row * a.parts * a.top;
#pragma unroll
    for (int e = 0; e < kEach; ++e) words[e] = e * 64 + lane < a.parts * a.top ? keys[e * 64 + lane] : 0;
    if (lane < a.parts) {
      const float4 p = a.sums[row * a.parts + lane];
      s = Sums{p.x, p.y, p.z};
    }
    s = JoinLanes<true>(s, a.factor);
    const float log_sum = LogSum(s);
    if (lane == 0) WriteRow<T>(a, s, log_sum, row);
    if (a.top == 0) continue;
    if (log_sum != log_sum) {
      if (lane < a.top) WriteTop(a, s, log_sum, row, lane, 0);
      continue;
    }
    // (keys differ from each other: a.top of them are no less than the least)
    const Key least = Least<kEach>(words, a.top);
    int before = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const unsigned long long found = __ballot(words[e] != 0 && words[e] >= least);
      const int place = before + __popcll(found & ((1ull << lane) - 1));
      if ((found >> lane & 1) && place < kMostTop) s_top[place] = words[e];
      before += __popcll(found);
    }
    __syncthreads();
    const Key mine = lane < a.top ? s_top[lane] : 0;
    int place = 0;
    for (int l = 0; l < a.top; ++l) place += LaneKey(mine, l) > mine;
    if (lane < a.top) WriteTop(a, s, log_sum, row, place, mine);
    __syncthreads();
  }
}

// ------------------------------------------------------------------ a row a thread

// The greatest kHeld in one pass, in order; `top` beyond that takes further passes, each behind the last one found.  kUnroll classes
// are asked for at once (kSide: side by side, in vectors).  Memory bounds it where the top is short: 1,000,003 x 10 fp32 class by class, top 3, 76 MB in 17.5 us, 4.3 TB/s.
template <typename T, bool kSide, int kHeld, int kUnroll>
__global__ void __launch_bounds__(256) k_columns(const RowsArgs a) {
  const long long step = (long long)gridDim.x * 256;
  for (long long row = (long long)blockIdx.x * 256 + threadIdx.x; row < a.n; row += step) {
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    Sums s = {-Infinity(), 0.0f, 0.0f};
    float log_sum = 0.0f, limit = Infinity();
    unsigned limit_at = 0;  // the last one found: what comes next is less, or as much and behind it
    for (int from = 0; from == 0 || from < a.top; from += kHeld) {
      float held[kHeld];  // (NaN: empty)
      unsigned held_at[kHeld];
#pragma unroll
      for (int h = 0; h < kHeld; ++h) held[h] = __builtin_nanf(""), held_at[h] = ~0u;
      for (unsigned j0 = 0; j0 < a.vocab; j0 += kUnroll) {
        float v[kUnroll];
        if (kSide && a.vocab - j0 >= kUnroll) {
          const Pack<T, kUnroll> p = *reinterpret_cast<const Pack<T, kUnroll> *>(x + j0);
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) v[u] = (float)p.v[u];
        } else {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) v[u] = (float)x[(long long)min(j0 + u, a.vocab - 1) * a.class_stride];
        }
        if (from == 0) {
          float most = v[0];
#pragma unroll
          for (int u = 1; u < kUnroll; ++u) most = fmaxf(most, v[u]);  // (the last class again, where there is no other)
          if (most > s.most) {
            const float d = a.factor * (s.most - most), e = Exp2(d);
            s.moment = e * (s.moment + fmaxf(d, kLowest) * s.sum);
            s.sum *= e;
            s.most = most;
          }
          const float base = Base(s.most);
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            if (j0 + u >= a.vocab) break;
            const float d = a.factor * (v[u] - base), e = Exp2(d);
            s.sum += e;
            s.moment = fmaf(fmaxf(d, kLowest), e, s.moment);
          }
        }
        if (a.top > 0) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            if (j0 + u >= a.vocab) break;
            float value = v[u];
            unsigned at = j0 + u;
            bool moves = false;
            if (from > 0 && !(value < limit || (value == limit && at > limit_at))) continue;
#pragma unroll
            for (int h = 0; h < kHeld; ++h) {  // (it takes its place before the first that is less, or empty, and those from there on move)
              moves = moves || !(value <= held[h]);
              const float other = held[h];
              const unsigned other_at = held_at[h];
              held[h] = moves ? value : other;
              held_at[h] = moves ? at : other_at;
              value = moves ? other : value;
              at = moves ? other_at : at;
            }
          }
        }
      }
      if (from == 0) {
        log_sum = LogSum(s);
        WriteRow<T>(a, s, log_sum, row);
      }
      if (kHeld == a.top) {  // (side by side)
        Pack<int, kHeld> tokens;
        Pack<float, kHeld> values;
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
          tokens.v[h] = log_sum != log_sum ? -1 : (int)held_at[h];
          values.v[h] = a.scale * (held[h] - Base(s.most)) - log_sum;
        }
        *reinterpret_cast<Pack<int, kHeld> *>(a.top_tokens + row * kHeld) = tokens;
        *reinterpret_cast<Pack<float, kHeld> *>(a.top_log_probs + row * kHeld) = values;
      } else {
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
          if (from + h < a.top) WriteTop(a, s, log_sum, row, from + h, held[h], held_at[h]);
      }
      limit = held[kHeld - 1];
      limit_at = held_at[kHeld - 1];
    }
  }
}

// ------------------------------------------------------------------ gradient

struct GradArgs {
  void *grad;
  const void *logits;
  long long row_stride, class_stride, grad_row_stride, grad_class_stride;
  long long n;
  unsigned vocab;
  float scale;
  const void *tokens;
  int token_bits;
  const float2 *stats;
  const float *grad_log_probs, *grad_entropy, *entropy;
  unsigned *status;
};

// A row's constants.  In powers of two, with d = log2 p,
//   grad_j = p_j (of_p + of_log d), and with [j = token] the one where p is taken from
struct RowGrad {
  float most, log_sum, of_p, of_log, weight, entropy;
  unsigned token;  // vocab for none
  bool live;       // false: a row of padding, whose gradient is 0 whatever its logits (and what they make of its sums)
};

template <bool kEntropy>
__device__ __forceinline__ RowGrad RowGradOf(const GradArgs &a, long long row) {
  RowGrad r;
  const float2 stats = a.stats[row];
  // (a row of nothing but minus infinity: whatever is subtracted from it, its powers are 0)
  const bool nothing = stats.x == -Infinity() && stats.y == 0.0f;
  r.most = nothing ? 0.0f : stats.x;
  r.log_sum = stats.y * kLog2E;
  const long long token = a.tokens == nullptr ? -1 : a.token_bits == 32 ? (long long)static_cast<const int *>(a.tokens)[row] : static_cast<const long long *>(a.tokens)[row];
  const bool there = token >= 0 && token < (long long)a.vocab;
  if (!there && token != -1 && a.status != nullptr) *a.status = 1u;
  r.token = there && !nothing ? (unsigned)token : a.vocab;
  r.weight = there ? a.scale * a.grad_log_probs[row] : 0.0f;
  if (nothing) r.weight = 0.0f;
  r.entropy = r.of_log = 0.0f;
  r.of_p = -r.weight;
  r.live = there;
  if (kEntropy) {
    const float h = nothing ? 0.0f : a.scale * a.grad_entropy[row];
    r.live = there || h != 0.0f;
    r.entropy = a.entropy[row];
    r.of_log = -h * kLn2;
    r.of_p -= h * r.entropy;
  }
  return r;
}

template <bool kEntropy>
__device__ __forceinline__ float GradOf(const RowGrad &r, float factor, float x) {
  const float d = fmaf(factor, x - r.most, -r.log_sum), p = Exp2(d);
  return kEntropy ? p * fmaf(r.of_log, fmaxf(d, kLowest), r.of_p) : p * r.of_p;
}
// The gradient of the token itself: weight (1 - p) as it stands, where its parts would meet with opposite signs.
template <bool kEntropy>
__device__ __forceinline__ float GradOfToken(const RowGrad &r, float factor, float x) {
  const float d = fmaf(factor, x - r.most, -r.log_sum), p = Exp2(d);
  float g = r.weight * (1.0f - p);
  if (kEntropy) g += p * fmaf(r.of_log, fmaxf(d, kLowest), r.of_p + r.weight);
  return g;
}

// Classes side by side: `lanes` threads of a workgroup take a row's piece of lanes * kVec * kUnroll classes.  4096 x 131,072 bf16, 2 GiB: 360 us, 6.0 TB/s.
// (The gradient may take the place of the logits: what a thread writes only it has read.)
template <typename T, int kUnroll, bool kEntropy, bool kPast>
__global__ void __launch_bounds__(256) k_grad_rows(const GradArgs a, int lanes, unsigned pieces) {
  constexpr int kVec = 16 / sizeof(T);
  const unsigned of = threadIdx.x / lanes, t = threadIdx.x % lanes, teams = 256 / lanes;
  const long long items = a.n * pieces;
  const float factor = a.scale * kLog2E;
  for (long long item = (long long)blockIdx.x * teams + of; item < items; item += (long long)gridDim.x * teams) {
    const long long row = pieces == 1 ? item : item / pieces;
    const unsigned begin = (unsigned)(item - row * pieces) * (unsigned)(lanes * kVec * kUnroll);
    const RowGrad r = RowGradOf<kEntropy>(a, row);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *grad = static_cast<T *>(a.grad) + row * a.grad_row_stride;
    const bool whole = a.vocab - begin >= (unsigned)(lanes * kVec * kUnroll);
    Pack<T, kVec> p[kUnroll];
    int held[kUnroll];
    const auto store = [&](int u, const Pack<T, kVec> &v) {
      T *to = grad + begin + (u * lanes + t) * kVec;
      if (held[u] == kVec) {
        if constexpr (kPast) StorePast(to, v);
        else *reinterpret_cast<Pack<T, kVec> *>(to) = v;
      } else {
#pragma unroll
        for (int c = 0; c < kVec; ++c)
          if (c < held[u]) to[c] = v.v[c];
      }
    };
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned at = begin + (u * lanes + t) * kVec;
      held[u] = whole ? kVec : at < a.vocab ? (int)min(a.vocab - at, (unsigned)kVec) : 0;
    }
    if (!r.live) {  // (written and not read: 4096 x 131,072 bf16, 30 % padding, 563 -> 522 us with the forward pass)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) store(u, Pack<T, kVec>{});
      continue;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned at = begin + (u * lanes + t) * kVec;
      if (held[u] == kVec) {
        p[u] = *reinterpret_cast<const Pack<T, kVec> *>(x + at);
      } else {
#pragma unroll
        for (int c = 0; c < kVec; ++c) p[u].v[c] = c < held[u] ? x[at + c] : T(0);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned at = begin + (u * lanes + t) * kVec, hit = r.token - at;
      T of_token = T(0);
      if (hit < (unsigned)kVec) {  // (one lane of a row)
        float v = 0.0f;
#pragma unroll
        for (int c = 0; c < kVec; ++c) v = hit == (unsigned)c ? (float)p[u].v[c] : v;
        of_token = Round<T>(GradOfToken<kEntropy>(r, factor, v));
      }
#pragma unroll
      for (int c = 0; c < kVec; ++c) p[u].v[c] = Round<T>(GradOf<kEntropy>(r, factor, (float)p[u].v[c]));
      if (hit < (unsigned)kVec) {
#pragma unroll
        for (int c = 0; c < kVec; ++c) p[u].v[c] = hit == (unsigned)c ? of_token : p[u].v[c];
      }
      store(u, p[u]);
    }
  }
}

// A row a thread, `part` classes of it (a multiple of kUnroll) by each row of workgroups.
constexpr unsigned kColumnsUnroll = 8;
template <typename T, bool kEntropy>
__global__ void __launch_bounds__(256) k_grad_columns(const GradArgs a, unsigned part) {
  constexpr unsigned kUnroll = kColumnsUnroll;
  const unsigned begin = blockIdx.y * part, end = min(a.vocab, begin + part);
  const long long step = (long long)gridDim.x * 256;
  const float factor = a.scale * kLog2E;
  for (long long row = (long long)blockIdx.x * 256 + threadIdx.x; row < a.n; row += step) {
    const RowGrad r = RowGradOf<kEntropy>(a, row);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *grad = static_cast<T *>(a.grad) + row * a.grad_row_stride;
    for (unsigned j0 = begin; j0 < end; j0 += kUnroll) {
      float v[kUnroll];
#pragma unroll
      for (unsigned u = 0; u < kUnroll; ++u) v[u] = (float)x[(long long)min(j0 + u, a.vocab - 1) * a.class_stride];
#pragma unroll
      for (unsigned u = 0; u < kUnroll; ++u) {
        if (j0 + u >= end) break;
        const float g = j0 + u == r.token ? GradOfToken<kEntropy>(r, factor, v[u]) : GradOf<kEntropy>(r, factor, v[u]);
        grad[(long long)(j0 + u) * a.grad_class_stride] = Round<T>(r.live ? g : 0.0f);
      }
    }
  }
}

// ------------------------------------------------------------------ the host

// Few rows are cut into parts, two workgroups for a CU, of 16 KB of bf16 at least (bf16, us: 1 x 131,072 top 20 in 16 parts 17.7, in 4 20.5, in 32 31.7, whose keys
// the join waits for; 100 x 131,072 top 5 in 5 parts 25.5, whole 28.2; 300 rows whole 32.0, in 3 parts 37.1).
int PartsOf(long long n, long long vocab) {
  if (n <= 0 || n >= 256) return 1;
  return (int)std::max<long long>(1, std::min({(long long)kMostParts, 512 / n, (vocab + kPart - 1) / kPart}));
}

void CheckSizes(long long n, long long vocab, int top) {
  if (n < 0 || n >= (1ll << 31)) throw std::runtime_error("bad number of rows");
  if (vocab < 1 || vocab >= (1ll << 31) - 65536) throw std::runtime_error("bad number of classes");
  if (top < 0 || top > kMostTop) throw std::runtime_error("top must be 0 to " + std::to_string(kMostTop));
  if (top > vocab) throw std::runtime_error("top is more than there are classes");
}

void CheckLogits(const Logits &l) {
  CheckType(l.type);
  CheckSizes(l.n, l.vocab, 0);
  if (l.row_stride < 0 || l.class_stride < 0) throw std::runtime_error("strides must not be negative");
  const long long most = (1ll << 62) / std::max<long long>(1, std::max(l.n, l.vocab));
  if (l.row_stride >= most / 2 || l.class_stride >= most / 2) throw std::runtime_error("strides are too large");
  if (!(l.scale > 0) || !std::isfinite(l.scale) || l.scale < std::numeric_limits<float>::min() || !std::isfinite(l.scale * kLog2E))
    throw std::runtime_error("scale must be a positive number within float32");
  if (l.tokens && l.token_bits != 32 && l.token_bits != 64) throw std::runtime_error("tokens must have 32 or 64 bits");
  if (l.n > 0 && !l.logits) throw std::runtime_error("null pointer argument");
  CheckAligned(l.logits, ElementBytes(l.type), "logits");
  if (l.tokens) CheckAligned(l.tokens, l.token_bits / 8, "tokens");
  CheckAligned(l.status, 4, "status");
}

unsigned GridOf(long long workgroups) { return (unsigned)std::min<long long>(workgroups, 1 << 20); }

}  // namespace

size_t LogProbsBytes(long long n, long long vocab, int top) {
  CheckSizes(n, vocab, top);
  const int parts = PartsOf(n, vocab);
  return parts == 1 ? 0 : (size_t)n * parts * (sizeof(float4) + (size_t)top * sizeof(Key));
}

void LogProbs(const LogProbsArgs &a) {
  const Logits &l = a.logits;
  CheckLogits(l);
  CheckSizes(l.n, l.vocab, a.top);
  if ((l.tokens == nullptr) != (a.log_probs == nullptr) && l.n > 0) throw std::runtime_error("tokens and log_probs go together");
  if (a.top > 0 && l.n > 0 && (!a.top_tokens || !a.top_log_probs)) throw std::runtime_error("null pointer argument");
  CheckAligned(a.log_probs, 4, "log_probs");
  CheckAligned(a.entropy, 4, "entropy");
  CheckAligned(a.stats, 8, "stats");
  CheckAligned(a.top_tokens, 4, "top_tokens");
  CheckAligned(a.top_log_probs, 4, "top_log_probs");
  const size_t need = LogProbsBytes(l.n, l.vocab, a.top);
  const bool side_by_side = l.class_stride == 1 || l.vocab == 1;
  if (need > 0) {
    if (!a.work) throw std::runtime_error("null pointer argument");
    CheckAligned(a.work, 16, "work");
    if (a.work_bytes < need) throw std::runtime_error("work memory is too small: " + std::to_string(need) + " bytes are needed");
  }
  if (l.n == 0) return;
  if (!a.log_probs && !a.entropy && !a.stats && a.top == 0) return;
  CheckApart({{a.log_probs, l.n * 4}, {a.entropy, l.n * 4}, {a.stats, l.n * 8}, {a.top_tokens, l.n * a.top * 4}, {a.top_log_probs, l.n * a.top * 4},
              {a.work, (long long)need}, {l.status, 4}},
             {Extent(l.logits, l.n, l.row_stride, l.vocab, l.class_stride, ElementBytes(l.type)), {l.tokens, l.n * l.token_bits / 8}});
  OnDeviceOf device(l.logits);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  RowsArgs r{l.logits, l.row_stride, l.class_stride, l.n, (unsigned)l.vocab, l.scale, l.scale * kLog2E, l.tokens, l.token_bits, a.log_probs,
             a.entropy, reinterpret_cast<float2 *>(a.stats), a.top, a.top_tokens, a.top_log_probs, l.status, 1, (unsigned)l.vocab, nullptr, nullptr};
  WithType(l.type, [&](auto type) {
    typedef decltype(type) T;
    // A thread a row where they are many for what each does, and where rows side by side are short enough for lines to stay in the L1; else teams (fp32, us, a thread
    // and teams: 64,000 x 10 top 5 14.9 and 55, 64,000 x 100 top 5 28 and 46, 16,000 x 100 top 5 25 and 14, 4000 x 100 top 20 92 and 14; 500,000 x 200
    // side by side 261 and 185).
    if ((!side_by_side || l.vocab <= 128) && l.n / 32 >= l.vocab * std::max(a.top, 1)) {
      const dim3 grid(GridOf((l.n + 255) / 256));
      const auto columns = [&](auto held) {
        if (side_by_side) hipLaunchKernelGGL((k_columns<T, true, decltype(held)::value, 8>), grid, dim3(256), 0, stream, r);
        else hipLaunchKernelGGL((k_columns<T, false, decltype(held)::value, 8>), grid, dim3(256), 0, stream, r);
      };
      // A list of each length to 8, whose rows are then stored side by side; longer ones eight at a time.  (1,000,003 x 10 fp32 class by class, us, by the next longer
      // list and by their own: top 4 26.8 and 24.5, top 6 36.6 and 27.8, top 7 44.9 and 29.4; top 8 31.)
      switch (std::min(a.top, 8)) {
        case 0:
        case 1: columns(std::integral_constant<int, 1>()); break;
        case 2: columns(std::integral_constant<int, 2>()); break;
        case 3: columns(std::integral_constant<int, 3>()); break;
        case 4: columns(std::integral_constant<int, 4>()); break;
        case 5: columns(std::integral_constant<int, 5>()); break;
        case 6: columns(std::integral_constant<int, 6>()); break;
        case 7: columns(std::integral_constant<int, 7>()); break;
        default: columns(std::integral_constant<int, 8>());
      }
      return;
    }
    r.parts = PartsOf(l.n, l.vocab);
    if (r.parts > 1) {
      r.part = (unsigned)((l.vocab + r.parts - 1) / r.parts + 7) / 8 * 8;
      r.parts = (int)((l.vocab + r.part - 1) / r.part);
      r.sums = static_cast<float4 *>(a.work);
      r.keys = reinterpret_cast<Key *>(r.sums + l.n * r.parts);
    }
    typedef std::true_type Yes;
    typedef std::false_type No;
    // A wave a row, or four.  One has no barriers, four have more on its way and keep the likeliest among more maxima (bf16, us, one and four:
    // 50,000 x 1000 top 10 63 and 294; 4000 x 8000 top 10 22 and 35, top 64 82 and 47; 4000 x 50,021 75 and 90, 1000 x 50,021 45 and 25; the parts of
    // 1 x 131,072 top 20 22 and 18).
    const size_t bytes = r.part * sizeof(T);
    const bool wave = r.parts == 1 && (a.top > 32 ? bytes <= 2048 : bytes <= 16384 || (bytes <= 65536 && a.top <= 5 && l.n >= 4096));
    const auto launch = [&](auto side, auto entropy, auto top) {
      constexpr bool kSide = decltype(side)::value, kEntropy = decltype(entropy)::value, kTop = decltype(top)::value;
      const long long items = l.n * r.parts;
      if (wave) hipLaunchKernelGGL((k_rows<T, 1, 2, kSide, kEntropy, kTop>), dim3(GridOf((items + 3) / 4)), dim3(256), 0, stream, r);
      else hipLaunchKernelGGL((k_rows<T, 4, 2, kSide, kEntropy, kTop>), dim3(GridOf(items)), dim3(256), 0, stream, r);
    };
    const auto launch_as = [&](auto side) {
      if (a.entropy && a.top) launch(side, Yes(), Yes());
      else if (a.entropy) launch(side, Yes(), No());
      else if (a.top) launch(side, No(), Yes());
      else launch(side, No(), No());
    };
    if (side_by_side) launch_as(Yes());
    else launch_as(No());
    if (r.parts > 1 && r.parts * r.top <= 512) hipLaunchKernelGGL((k_join<T, 8>), dim3(GridOf(l.n)), dim3(64), 0, stream, r);
    else if (r.parts > 1) hipLaunchKernelGGL((k_join<T, 32>), dim3(GridOf(l.n)), dim3(64), 0, stream, r);
  });
  HIP_OK(hipGetLastError());
}

void LogProbsGrad(const LogProbsGradArgs &a) {
  const Logits &l = a.logits;
  CheckLogits(l);
  if (a.grad_row_stride < 0 || a.grad_class_stride < 0) throw std::runtime_error("strides must not be negative");
  const long long most = (1ll << 62) / std::max<long long>(1, std::max(l.n, l.vocab));
  if (a.grad_row_stride >= most / 2 || a.grad_class_stride >= most / 2) throw std::runtime_error("strides are too large");
  if (l.n == 0) return;
  // two elements of the gradient must not share a place
  const bool rows_apart = l.n == 1 || a.grad_row_stride >= 1, classes_apart = l.vocab == 1 || a.grad_class_stride >= 1;
  const bool apart = l.n == 1 || l.vocab == 1 || a.grad_row_stride >= (l.vocab - 1) * a.grad_class_stride + 1 ||
                     a.grad_class_stride >= (l.n - 1) * a.grad_row_stride + 1;
  if (!rows_apart || !classes_apart || !apart) throw std::runtime_error("rows of the gradient overlap");
  if (!a.grad_logits || !a.stats) throw std::runtime_error("null pointer argument");
  if ((l.tokens == nullptr) != (a.grad_log_probs == nullptr)) throw std::runtime_error("tokens and grad_log_probs go together");
  if ((a.grad_entropy == nullptr) != (a.entropy == nullptr)) throw std::runtime_error("grad_entropy and entropy go together");
  if (a.grad_logits == l.logits && ((l.n > 1 && a.grad_row_stride != l.row_stride) || (l.vocab > 1 && a.grad_class_stride != l.class_stride)))
    throw std::runtime_error("a gradient in the place of the logits has their strides");
  CheckAligned(a.grad_logits, ElementBytes(l.type), "grad_logits");
  CheckAligned(a.grad_log_probs, 4, "grad_log_probs");
  CheckAligned(a.grad_entropy, 4, "grad_entropy");
  CheckAligned(a.entropy, 4, "entropy");
  CheckAligned(a.stats, 8, "stats");
  const Extent none(nullptr, 0), grad = Extent(a.grad_logits, l.n, a.grad_row_stride, l.vocab, a.grad_class_stride, ElementBytes(l.type));
  CheckApart({grad, {l.status, 4}},
             {a.grad_logits == l.logits ? none : Extent(l.logits, l.n, l.row_stride, l.vocab, l.class_stride, ElementBytes(l.type)), {l.tokens, l.n * l.token_bits / 8}, {a.stats, l.n * 8},
              {a.grad_log_probs, l.n * 4}, {a.grad_entropy, l.n * 4}, {a.entropy, l.n * 4}});
  OnDeviceOf device(a.grad_logits);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  const GradArgs g{a.grad_logits, l.logits, l.row_stride, l.class_stride, a.grad_row_stride, a.grad_class_stride, l.n, (unsigned)l.vocab, l.scale,
                   l.tokens, l.token_bits, reinterpret_cast<const float2 *>(a.stats), a.grad_log_probs, a.grad_entropy, a.entropy, l.status};
  const bool side_by_side = l.vocab == 1 || (l.class_stride == 1 && a.grad_class_stride == 1);
  WithType(l.type, [&](auto type) {
    typedef decltype(type) T;
    const auto launch = [&](auto entropy) {
      constexpr bool kEntropy = decltype(entropy)::value;
      if (!side_by_side) {
        // few rows share out their classes, at least 64 to a part, until there are threads for the chip
        const long long parts = std::max(1ll, std::min({(1ll << 18) / l.n, l.vocab / 64, 32768ll}));
        const unsigned part = (unsigned)((l.vocab + parts - 1) / parts + kColumnsUnroll - 1) / kColumnsUnroll * kColumnsUnroll;
        hipLaunchKernelGGL((k_grad_columns<T, kEntropy>), dim3(GridOf((l.n + 255) / 256), (unsigned)((l.vocab + part - 1) / part)), dim3(256), 0, stream, g, part);
        return;
      }
      // threads of a row, or of as much of one as a workgroup takes: vectors of up to 32 threads one each, or four each (1,000,003 x 10 fp32 with the forward pass
      // 39 us, with four a thread, which is a row a thread, 57)
      const auto rows = [&](auto unroll, auto past) {
        constexpr int kUnroll = decltype(unroll)::value, kEach = 16 / sizeof(T) * kUnroll;
        int lanes = kUnroll == 1 ? 32 : 256;
        while (lanes > 1 && lanes / 2 * kEach >= l.vocab) lanes /= 2;
        const unsigned pieces = (unsigned)((l.vocab + lanes * kEach - 1) / (lanes * kEach));
        const long long items = l.n * pieces, teams = 256 / lanes;
        hipLaunchKernelGGL((k_grad_rows<T, kUnroll, kEntropy, decltype(past)::value>), dim3(GridOf((items + teams - 1) / teams)), dim3(256), 0, stream, g, lanes, pieces);
      };
      const auto rows_of = [&](auto past) {
        if (l.vocab <= 32 * 16 / (long long)sizeof(T)) rows(std::integral_constant<int, 1>(), past);
        else rows(std::integral_constant<int, 4>(), past);
      };
      // a gradient that the L2 caches do not hold is written past them (4096 x 131,072 bf16: 491 us through them, 358 past)
      if ((size_t)l.n * l.vocab * sizeof(T) > kStreamedBytes) rows_of(std::true_type());
      else rows_of(std::false_type());
    };
    if (a.grad_entropy) launch(std::true_type());
    else launch(std::false_type());
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
