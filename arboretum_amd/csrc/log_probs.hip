// Log probabilities of given tokens under rows of logits, the entropy of each row, its likeliest tokens, and the gradient
// of the logits.  With a_j = scale (x_j - max x) and S = sum exp a_j,
//   log_prob = a_token - log S,   entropy = log S - (sum a_j exp a_j) / S,
//   grad_j   = scale (g ([j = token] - p_j) - h p_j (log p_j + entropy)),   p_j = exp(a_j - log S).
// A row is read once: maximum, S and sum a exp a run along it, and a new maximum scales what was summed before
// (sum (a + d) exp (a + d) = exp d (sum a exp a + d sum exp a)).
#include <algorithm>
#include <cmath>
#include <limits>

#include "operators_device.h"

namespace arb {
namespace {

typedef unsigned long long Key;  // value (in an order of whole numbers) and inverted index: the greater one comes first; 0: none

constexpr int kMostTop = 64;     // of them a wave holds one a lane
constexpr int kMostParts = 64;   // of a row, joined by a wave
constexpr long long kPart = 2048;  // a row is not cut into less
constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLowest = -1.0e20f;  // exponents beyond are taken for it where they are factors: their power is 0, and must not meet an infinity

__device__ __forceinline__ float Infinity() { return __builtin_inff(); }
__device__ __forceinline__ float Exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ Key KeyOf(float value, unsigned index) {
  const unsigned bits = __float_as_uint(value + 0.0f);  // (-0 and 0 are equal)
  const unsigned order = bits ^ ((bits >> 31) ? 0xFFFFFFFFu : 0x80000000u);
  return ((Key)order << 32) | (Key)(~index);
}
__device__ __forceinline__ float ValueOf(Key key) {
  const unsigned order = (unsigned)(key >> 32);
  return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ unsigned IndexOf(Key key) { return ~(unsigned)key; }

__device__ __forceinline__ Key LaneKey(Key key, int lane) {
  const unsigned low = __builtin_amdgcn_readlane((int)(unsigned)key, lane), high = __builtin_amdgcn_readlane((int)(unsigned)(key >> 32), lane);
  return ((Key)high << 32) | low;
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
    const float h = s.sum == 0.0f ? 0.0f : log_sum - 0.693147180559945309f * (s.moment / s.sum);
    a.entropy[i] = h;
  }
  if (a.stats != nullptr) a.stats[i] = make_float2(s.most, log_sum);
}

__device__ __forceinline__ void WriteTop(const RowsArgs &a, const Sums &s, float log_sum, long long i, int rank, Key key) {
  const bool none = log_sum != log_sum;  // a row with a NaN, or plus infinity
  a.top_tokens[i * a.top + rank] = none ? -1 : (int)IndexOf(key);
  a.top_log_probs[i * a.top + rank] = a.scale * (ValueOf(key) - Base(s.most)) - log_sum;
}

// ------------------------------------------------------------------ rows whose classes lie side by side

// A team of kWaves waves reads a row, or a part of one; one wave a row: four teams a workgroup.
// Every thread keeps the maximum of what it reads.  Of the whole row the k likeliest can only be where the k greatest of
// these maxima are (whoever is in no such thread is behind k others), so only those threads' share of the row is read again.
template <typename T, int kWaves, int kUnroll, bool kEntropy, bool kTop>
__global__ void __launch_bounds__(kWaves == 1 ? 256 : kWaves * 64) k_rows(const RowsArgs a) {
  constexpr int kVec = 16 / sizeof(T), kTeam = kWaves * 64, kTeams = kWaves == 1 ? 4 : 1, kChunk = kUnroll * kVec;
  __shared__ Sums s_sums[kWaves];
  __shared__ Key s_lists[kTop ? kTeams * kWaves : 1][kTop ? kMostTop : 1];
  __shared__ Key s_top[kTop ? kTeams : 1][kTop ? kMostTop : 1];
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
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride + begin;

    Sums s = {-Infinity(), 0.0f, 0.0f};
    unsigned best = 0;  // vector from which on the maximum is found
    const auto add = [&](const float (&v)[kChunk], unsigned at) {
      float most = v[0];
#pragma unroll
      for (int c = 1; c < kChunk; ++c) most = fmaxf(most, v[c]);
      if (most > s.most) {
        if (kTop) best = at;
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
      for (int u = 0; u < kUnroll; ++u) p[u] = *reinterpret_cast<const Pack<T, kVec> *>(x + (size_t)((i + u) * kTeam + t) * kVec);
      float v[kChunk];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int c = 0; c < kVec; ++c) v[u * kVec + c] = (float)p[u].v[c];
      add(v, i);
    }
    if ((size_t)whole * kTeam + t < vectors) {  // the rest; what is beyond the end counts as minus infinity
      float v[kChunk];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const unsigned at = ((whole + u) * kTeam + t) * kVec;
        const bool all = at < length && length - at >= kVec;
        Pack<T, kVec> p;
        if (all) p = *reinterpret_cast<const Pack<T, kVec> *>(x + at);
#pragma unroll
        for (int c = 0; c < kVec; ++c) v[u * kVec + c] = all ? (float)p.v[c] : at < length && c < (int)(length - at) ? (float)x[at + c] : -Infinity();
      }
      add(v, whole);
    }
    // the thread's greatest value, the first of equal ones
    Key mine = 0;
    if (kTop && t < vectors) {
      for (unsigned i = best, end = best + kUnroll; i < end && mine == 0; ++i) {
        const unsigned at = (i * kTeam + t) * kVec;
        for (int c = 0; c < kVec; ++c)
          if (mine == 0 && at < length && (unsigned)c < length - at && (float)x[at + c] == s.most) mine = KeyOf(s.most, begin + at + c);
      }
    }

    // the sums of the team
#pragma unroll
    for (int by = 32; by > 0; by /= 2) s = Join(s, Sums{__shfl_xor(s.most, by), __shfl_xor(s.sum, by), __shfl_xor(s.moment, by)}, a.factor);
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
      // Ranks: how many keys of the wave are greater, then how many of each other wave's list.
      Key(*lists)[kMostTop] = &s_lists[team * kWaves];
      const auto rank = [&](Key key, Key *to) {  // the team's greatest a.top keys to `to`, in order; whatever else there is: 0
        int r = 0;
        for (int l = 0; l < 64; ++l) {
          const Key other = LaneKey(key, l);
          r += other > key || (other == key && l < lane);
        }
        if (kWaves == 1) {
          if (r < a.top) to[r] = key;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
          __builtin_amdgcn_wave_barrier();
          return;
        }
        lists[wave][r] = key;
        __syncthreads();
        int all = r;
        if (r < a.top && key != 0) {
          for (int w = 0; w < kWaves; ++w) {
            if (w == wave) continue;
            int low = 0, high = kMostTop;  // keys before `low` are greater, those from `high` on are not
            while (low < high) {
              const int mid = (low + high) / 2;
              if (lists[w][mid] > key) low = mid + 1;
              else high = mid;
            }
            all += low;
          }
          if (all < a.top) to[all] = key;
        }
        __syncthreads();
      };
      if (t < kMostTop) s_top[team][t] = 0;
      if (kWaves > 1) __syncthreads();
      rank(mine, s_top[team]);
      const Key least = s_top[team][a.top - 1];
      Key held = 0;  // of the wave, a sorted list, one a lane
      for (int k = wave; k < a.top; k += kWaves) {
        const Key owner = s_top[team][k];
        if (owner == 0) break;
        const unsigned from = (IndexOf(owner) - begin) / kVec % kTeam;
        const unsigned rounds = (vectors - from + kTeam - 1) / kTeam;
        for (unsigned e = lane; e - lane < rounds * kVec; e += 64) {
          const unsigned at = (e / kVec * kTeam + from) * kVec + e % kVec;
          const Key key = e < rounds * kVec && at < length ? KeyOf((float)x[at], begin + at) : 0;
          unsigned long long found = __ballot(key != 0 && key >= least);
          while (found != 0) {
            const Key one = LaneKey(key, __builtin_ctzll(found));
            found &= found - 1;
            const int place = __popcll(__ballot(held > one));
            const Key before = ((Key)(unsigned)__shfl_up((int)(unsigned)(held >> 32), 1) << 32) | (unsigned)__shfl_up((int)(unsigned)held, 1);
            held = lane < place ? held : lane == place ? one : before;
          }
        }
      }
      if (kWaves > 1) __syncthreads();
      if (t < kMostTop) s_top[team][t] = 0;
      if (kWaves > 1) __syncthreads();
      rank(held, s_top[team]);
      if (live && (int)t < a.top) {
        if (a.parts == 1) WriteTop(a, s, log_sum, row, t, s_top[team][t]);
        else a.keys[item * a.top + t] = s_top[team][t];
      }
    }
    if (kWaves > 1) __syncthreads();
  }
}

// The parts of a row, by one wave: a lane holds a part.
template <typename T>
__global__ void __launch_bounds__(64) k_join(const RowsArgs a) {
  const int lane = threadIdx.x;
  for (long long row = blockIdx.x; row < a.n; row += gridDim.x) {
    Sums s = {-Infinity(), 0.0f, 0.0f};
    if (lane < a.parts) {
      const float4 p = a.sums[row * a.parts + lane];
      s = Sums{p.x, p.y, p.z};
    }
#pragma unroll
    for (int by = 32; by > 0; by /= 2) s = Join(s, Sums{__shfl_xor(s.most, by), __shfl_xor(s.sum, by), __shfl_xor(s.moment, by)}, a.factor);
    const float log_sum = LogSum(s);
    if (lane == 0) WriteRow<T>(a, s, log_sum, row);
    const Key *keys = a.keys + (row * a.parts + lane) * a.top;
    int at = 0;  // the heads of the parts' lists; the greatest leaves its list
    Key head = lane < a.parts && a.top > 0 ? keys[0] : 0;
    for (int k = 0; k < a.top; ++k) {
      Key most = head;
#pragma unroll
      for (int by = 32; by > 0; by /= 2) {
        const Key other = ((Key)(unsigned)__shfl_xor((int)(unsigned)(most >> 32), by) << 32) | (unsigned)__shfl_xor((int)(unsigned)most, by);
        most = max(most, other);
      }
      if (lane == 0) WriteTop(a, s, log_sum, row, k, most);
      if (head == most && lane < a.parts) head = ++at < a.top ? keys[at] : 0;
    }
  }
}

// ------------------------------------------------------------------ a row a thread

// The greatest kHeld in one pass, in order; `top` beyond that takes further passes, each behind the last one found.
template <typename T, int kHeld>
__global__ void __launch_bounds__(256) k_columns(const RowsArgs a) {
  constexpr int kUnroll = 4;
  const long long step = (long long)gridDim.x * 256;
  for (long long row = (long long)blockIdx.x * 256 + threadIdx.x; row < a.n; row += step) {
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    Sums s = {-Infinity(), 0.0f, 0.0f};
    float log_sum = 0.0f;
    Key limit = ~0ull;
    for (int from = 0; from == 0 || from < a.top; from += kHeld) {
      Key held[kHeld];
#pragma unroll
      for (int h = 0; h < kHeld; ++h) held[h] = 0;
      for (unsigned j0 = 0; j0 < a.vocab; j0 += kUnroll) {
        float v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = j0 + u < a.vocab ? (float)x[(long long)min(j0 + u, a.vocab - 1) * a.class_stride] : -Infinity();
        if (from == 0) {
          float most = s.most;
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) most = fmaxf(most, v[u]);
          if (most > s.most) {
            const float d = a.factor * (s.most - most), e = Exp2(d);
            s.moment = e * (s.moment + fmaxf(d, kLowest) * s.sum);
            s.sum *= e;
            s.most = most;
          }
          const float base = Base(s.most);
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            const float d = a.factor * (v[u] - base), e = Exp2(d);
            s.sum += e;
            s.moment = fmaf(fmaxf(d, kLowest), e, s.moment);
          }
        }
        if (a.top > 0) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            Key key = KeyOf(v[u], j0 + u);
            if (j0 + u >= a.vocab || key >= limit) key = 0;
#pragma unroll
            for (int h = 0; h < kHeld; ++h) {  // (in order: it takes its place, those behind move on)
              const Key lower = min(held[h], key);
              held[h] = max(held[h], key);
              key = lower;
            }
          }
        }
      }
      if (from == 0) {
        log_sum = LogSum(s);
        WriteRow<T>(a, s, log_sum, row);
      }
#pragma unroll
      for (int h = 0; h < kHeld; ++h)
        if (from + h < a.top) WriteTop(a, s, log_sum, row, from + h, held[h]);
      limit = held[kHeld - 1];
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

// A row's constants.
struct RowGrad {
  float most, log_sum, weight, entropy_weight, entropy;
  long long token;
  bool nothing;  // no logit but minus infinity: no gradient
};

__device__ __forceinline__ RowGrad RowGradOf(const GradArgs &a, long long row) {
  RowGrad r;
  const float2 stats = a.stats[row];
  r.most = stats.x;
  r.log_sum = stats.y;
  r.nothing = stats.x == -Infinity() && stats.y == 0.0f;
  r.token = a.tokens == nullptr ? -1 : a.token_bits == 32 ? (long long)static_cast<const int *>(a.tokens)[row] : static_cast<const long long *>(a.tokens)[row];
  if (r.token < 0 || r.token >= (long long)a.vocab) {
    if (r.token != -1 && a.status != nullptr) *a.status = 1u;
    r.token = -1;
  }
  r.weight = r.token >= 0 ? a.grad_log_probs[row] : 0.0f;
  r.entropy_weight = a.grad_entropy != nullptr ? a.grad_entropy[row] : 0.0f;
  r.entropy = a.grad_entropy != nullptr ? a.entropy[row] : 0.0f;
  return r;
}

template <typename T>
__device__ __forceinline__ T GradOf(const GradArgs &a, const RowGrad &r, float x, long long j) {
  const float log_p = a.scale * (x - r.most) - r.log_sum;
  const float p = Exp2(log_p * kLog2E);
  float g = r.weight * ((j == r.token ? 1.0f : 0.0f) - p);
  if (a.grad_entropy != nullptr) g -= r.entropy_weight * (p > 0.0f ? p * (log_p + r.entropy) : p);
  return Round<T>(r.nothing ? 0.0f : a.scale * g);
}

// Classes side by side: `lanes` threads of a workgroup take a row's piece of lanes * kVec * kUnroll classes.
// (The gradient may take the place of the logits: what a thread writes only it has read.)
template <typename T, int kUnroll>
__global__ void __launch_bounds__(256) k_grad_rows(const GradArgs a, int lanes, unsigned pieces) {
  constexpr int kVec = 16 / sizeof(T);
  const unsigned of = threadIdx.x / lanes, t = threadIdx.x % lanes, teams = 256 / lanes;
  const long long items = a.n * pieces;
  for (long long item = (long long)blockIdx.x * teams + of; item < items; item += (long long)gridDim.x * teams) {
    const long long row = pieces == 1 ? item : item / pieces;
    const unsigned begin = (unsigned)(item - row * pieces) * (unsigned)(lanes * kVec * kUnroll);
    const RowGrad r = RowGradOf(a, row);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *grad = static_cast<T *>(a.grad) + row * a.grad_row_stride;
    if (a.vocab - begin >= (unsigned)(lanes * kVec * kUnroll)) {
      Pack<T, kVec> p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = *reinterpret_cast<const Pack<T, kVec> *>(x + begin + (u * lanes + t) * kVec);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const unsigned at = begin + (u * lanes + t) * kVec;
#pragma unroll
        for (int c = 0; c < kVec; ++c) p[u].v[c] = GradOf<T>(a, r, (float)p[u].v[c], at + c);
        *reinterpret_cast<Pack<T, kVec> *>(grad + at) = p[u];
      }
    } else {
      for (unsigned at = begin + t; at < a.vocab; at += lanes) grad[at] = GradOf<T>(a, r, (float)x[at], at);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_grad_columns(const GradArgs a) {
  constexpr int kUnroll = 4;
  const long long step = (long long)gridDim.x * 256;
  for (long long row = (long long)blockIdx.x * 256 + threadIdx.x; row < a.n; row += step) {
    const RowGrad r = RowGradOf(a, row);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *grad = static_cast<T *>(a.grad) + row * a.grad_row_stride;
    for (unsigned j0 = 0; j0 < a.vocab; j0 += kUnroll) {
      float v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = (float)x[(long long)min(j0 + u, a.vocab - 1) * a.class_stride];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j0 + u < a.vocab) grad[(long long)(j0 + u) * a.grad_class_stride] = GradOf<T>(a, r, v[u], j0 + u);
    }
  }
}

// ------------------------------------------------------------------ the host

// Few rows are cut into parts that fill the chip.
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
  OnDeviceOf device(l.logits);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  RowsArgs r{l.logits, l.row_stride, l.class_stride, l.n, (unsigned)l.vocab, l.scale, l.scale * kLog2E, l.tokens, l.token_bits, a.log_probs,
             a.entropy, reinterpret_cast<float2 *>(a.stats), a.top, a.top_tokens, a.top_log_probs, l.status, 1, (unsigned)l.vocab, nullptr, nullptr};
  WithType(l.type, [&](auto type) {
    typedef decltype(type) T;
    if (!side_by_side || l.vocab <= 32) {
      const unsigned grid = GridOf((l.n + 255) / 256);
      if (a.top <= 4) hipLaunchKernelGGL((k_columns<T, 4>), dim3(grid), dim3(256), 0, stream, r);
      else hipLaunchKernelGGL((k_columns<T, 8>), dim3(grid), dim3(256), 0, stream, r);
      return;
    }
    r.parts = PartsOf(l.n, l.vocab);
    if (r.parts > 1) {
      r.part = (unsigned)((l.vocab + r.parts - 1) / r.parts + 7) / 8 * 8;
      r.parts = (int)((l.vocab + r.part - 1) / r.part);
      r.sums = static_cast<float4 *>(a.work);
      r.keys = reinterpret_cast<Key *>(r.sums + l.n * r.parts);
    }
    const auto launch = [&](auto entropy, auto top) {
      constexpr bool kEntropy = decltype(entropy)::value, kTop = decltype(top)::value;
      const long long items = l.n * r.parts;
      if (r.parts > 1) hipLaunchKernelGGL((k_rows<T, 4, 1, kEntropy, kTop>), dim3(GridOf(items)), dim3(256), 0, stream, r);
      else if (r.part <= 2048) hipLaunchKernelGGL((k_rows<T, 1, 1, kEntropy, kTop>), dim3(GridOf((items + 3) / 4)), dim3(256), 0, stream, r);
      else hipLaunchKernelGGL((k_rows<T, 4, 4, kEntropy, kTop>), dim3(GridOf(items)), dim3(256), 0, stream, r);
    };
    typedef std::true_type Yes;
    typedef std::false_type No;
    if (a.entropy && a.top) launch(Yes(), Yes());
    else if (a.entropy) launch(Yes(), No());
    else if (a.top) launch(No(), Yes());
    else launch(No(), No());
    if (r.parts > 1) hipLaunchKernelGGL((k_join<T>), dim3(GridOf(l.n)), dim3(64), 0, stream, r);
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
  OnDeviceOf device(a.grad_logits);
  const hipStream_t stream = static_cast<hipStream_t>(a.stream);
  const GradArgs g{a.grad_logits, l.logits, l.row_stride, l.class_stride, a.grad_row_stride, a.grad_class_stride, l.n, (unsigned)l.vocab, l.scale,
                   l.tokens, l.token_bits, reinterpret_cast<const float2 *>(a.stats), a.grad_log_probs, a.grad_entropy, a.entropy, l.status};
  const bool side_by_side = l.vocab == 1 || (l.class_stride == 1 && a.grad_class_stride == 1);
  WithType(l.type, [&](auto type) {
    typedef decltype(type) T;
    if (!side_by_side) {
      hipLaunchKernelGGL((k_grad_columns<T>), dim3(GridOf((l.n + 255) / 256)), dim3(256), 0, stream, g);
      return;
    }
    constexpr int kUnroll = 4, kVec = 16 / sizeof(T);
    int lanes = 256;
    while (lanes > 4 && lanes / 2 >= l.vocab) lanes /= 2;
    const unsigned pieces = (unsigned)((l.vocab + lanes * kVec * kUnroll - 1) / (lanes * kVec * kUnroll));
    const long long items = l.n * pieces, teams = 256 / lanes;
    hipLaunchKernelGGL((k_grad_rows<T, kUnroll>), dim3(GridOf((items + teams - 1) / teams)), dim3(256), 0, stream, g, lanes, pieces);
  });
  HIP_OK(hipGetLastError());
}

}  // namespace arb
