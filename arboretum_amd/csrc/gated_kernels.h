// A gated layer and its gradient.  With g = x Wg^T, u = x Wu^T (weights [hidden][dim]),
//   out = act(g) u,  silu(g) = g / (1 + e^-g),  gelu(g) = g Phi(g);
//   dg = grad u act'(g),  du = grad act(g),  grad_x = dg Wg + du Wu,  grad_Wg = dg^T x,  grad_Wu = du^T x.
// Products by matrix instructions, their sums in 32 bits.
#ifndef ARBORETUM_AMD_GATED_KERNELS_H_
#define ARBORETUM_AMD_GATED_KERNELS_H_
#include <algorithm>
#include <type_traits>
#include <utility>

#include "checkpoint.h"
#include "gated_launch.h"
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

// (the instructions for powers of two and reciprocals, of a rounding each: a division and expf take three times the time, and an
// epilogue of nothing but them is what bounds narrow layers.  Below -87.3, where 1 + e^-g passes 2^126, the reciprocal is 0: silu is 0 there instead of what is less than
// 2^-119)
__device__ __forceinline__ float PowerOfE(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
__device__ __forceinline__ float Sigmoid(float g) { return __builtin_amdgcn_rcpf(1.0f + PowerOfE(-g)); }

// Phi(g), and e^(-g^2/2) in two factors (which reach below 2^-126 together).  From -|g| on it is e^(-g^2/2) times Mills' ratio, here t P(t) with
// t = 1 / (1 + 0.35 |g|): P has the least greatest relative error that a polynomial of its degree has for 0 <= |g| <= 16 (3e-8, 9e-8 with its coefficients in 32 bits; summed in 32 bits 4e-7),
// beyond which the other factor is 0.  (erfcf has a branch for either end, of which a wave runs both: 1003 x 771 x 2055 took 20.2 us.)
__device__ __forceinline__ float Phi(float g, float *root) {
  const float a = fminf(fabsf(g), 16.0f), t = __builtin_amdgcn_rcpf(1.0f + 0.35f * a);
  constexpr float kP[9] = {0.13962124f, 0.13986452f, 0.11981419f, 0.10557979f, -0.023275260f, 0.15940905f, -0.25591564f, 0.14406730f, -0.029165233f};
  float p = kP[8];
#pragma unroll
  for (int n = 7; n >= 0; --n) p = fmaf(p, t, kP[n]);
  *root = __builtin_amdgcn_exp2f(-0.36067376022224085f * (a * a));
  const float tail = *root * (p * t) * *root;
  return g < 0.0f ? tail : 1.0f - tail;
}

template <int kAct>
__device__ __forceinline__ float Act(float g) {
  if (kAct == kSilu) return g * Sigmoid(g);
  float root;
  return g * Phi(g, &root);
}

// act(g) and act'(g)
template <int kAct>
__device__ __forceinline__ void ActAndSlope(float g, float *act, float *slope) {
  if (kAct == kSilu) {
    const float s = Sigmoid(g);
    *act = g * s;
    *slope = s + *act * (1.0f - s);
  } else {
    float root;
    const float phi = Phi(g, &root);
    *act = g * phi;
    *slope = phi + g * (0.39894228040143268f * root * root);
  }
}

// ------------------------------------------------------------------ matrix products

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
  const float *undo;       // what sums are multiplied with (a power of two), float16 only; may be null
};
template <typename T>
__device__ __forceinline__ float UndoOf(const Products &p) {
  return std::is_same_v<T, _Float16> && p.undo != nullptr ? *p.undo : 1.0f;
}

constexpr unsigned kNowhere = 0x80000000u;  // offset beyond every operand: a load from there gives 0

typedef int I4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char LdsByte;
typedef __attribute__((address_space(3))) I4 LdsI4;

// 16 bytes a lane from `base` + `at` (beyond 2^31: 0) to the LDS, the wave's 1 KB side by side from `to` + kOffset on.  By hand: the
// compiler waits for a load of its own before any read of the LDS, and this one is meant to be on its way meanwhile.  Whoever reads
// what it writes waits for it first (WaitAndMeet, which nothing that touches memory moves across).
// (The compiler itself keeps nothing in m0, and says so of the clobber; where it passes an index there, nothing of this comes in between.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int kOffset>
__device__ __forceinline__ void LoadToLds(unsigned long long base, unsigned at, unsigned to) {
  const I4 from = {(int)(unsigned)base, (int)(unsigned)(base >> 32), 0x7FFFFFFF, 0x00020000};
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(at), "s"(from), "s"(to), "n"(kOffset) : "m0", "scc");
}
#pragma clang diagnostic pop

// Until no more than kLast of the wave's loads are on their way (they arrive in the order they were issued in), what it has read of the LDS is there,
// and all waves of the workgroup are as far.
template <int kLast>
__device__ __forceinline__ void WaitAndMeet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLast) : "memory");
}

__device__ __forceinline__ void WaitForLoads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void Meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The chunks of an operand's block in the LDS.  Along k: line by line, 8 chunks each; across: k by k, the chunks of all lines.
// Chunks change places from line to line (from k to k), so that the lanes that read together meet other banks: they
// read one chunk of 16 lines, of which two make up all banks; or 32 bytes (16 lines of 16 bits) of eight k's, 64 bytes of four k's of 32 bits.
template <typename T, int kLines, bool kAcross>
struct Layout {
  static constexpr int kVec = 16 / sizeof(T), kRowChunks = kAcross ? kLines / kVec : 8;
  static constexpr int kReads = kAcross ? sizeof(T) : 1;  // of the LDS for a chunk of a product
  static __device__ __forceinline__ int Swap(int row) {
    if (!kAcross) return (row >> 1) & 7;
    if (sizeof(T) == 2) return (((row & 3) | ((row >> 1) & 4)) << 1) & (kRowChunks - 1);
    return (row & 12) & (kRowChunks - 1);
  }
  static __device__ __forceinline__ int At(int row, int chunk) { return (row * kRowChunks + (chunk ^ Swap(row))) * 16; }
  // The chunk of a product for line `line` (of lane % 16) and the quarter `quarter` of the k's of half `half`.
  static __device__ __forceinline__ Chunk<T> Read(const LdsByte *block, int first, int half) {
    const int lane = threadIdx.x & 63, quarter = lane / 16, l = lane % 16;
    if constexpr (!kAcross) {
      return __builtin_bit_cast(Chunk<T>, *(const LdsI4 *)(block + At(first + l, half * 4 + quarter)));
    } else if constexpr (sizeof(T) == 2) {
      // (16 lanes name the 8-byte pieces of four k's by 16 lines, and each gets the four k's of one line)
      typedef short S4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) S4 LdsS4;
      const int k = half * 32 + quarter * 8 + l / 4, chunk = first / 8 + l % 4 / 2, in = l % 2 * 8;
      const S4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4 *)(block + At(k, chunk) + in));
      const S4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4 *)(block + At(k + 4, chunk) + in));
      struct Both {
        S4 low, high;
      };
      return __builtin_bit_cast(Chunk<T>, (Both{low, high}));
    } else {
      Chunk<T> c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c.v[e] = *(const __attribute__((address_space(3))) float *)(block + At(half * 16 + quarter * 4 + e, (first + l) / 4) + (first + l) % 4 * 4);
      return c;
    }
  }
};

__device__ __forceinline__ unsigned long long Uniform(unsigned long long v) {
  return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)v);
}

// The k's of a tile's lines that lie one after the other: `blocks` blocks of them from `base` on (kPaired: 64 lines from there, 64 from `second`, the next
// 64 of each ...), `left` k's and `lines` lines (of each) from there to the operand's end.
struct Run {
  const void *base, *second;
  long long lines, left;
  int blocks;
};

// The row of a block's line (k, across): kPaired, of the gate or of up.
template <bool kPaired>
__device__ __forceinline__ int RowOf(int line) {
  return kPaired ? line / 128 * 64 + line % 64 : line;
}

// Which tiles a workgroup takes: `first`, and every `of`th from there.
struct Share {
  unsigned first, of;
};

// An operand's blocks, run after run and tile after tile, each by loads that write to the LDS: for operands whose chunks are aligned and
// whole.  A block costs its loads and next to nothing else: where a lane reads is worked out once a run.
template <typename T, int kLines, int kThreads, bool kAcross, bool kPaired>
struct Stream {
  typedef Layout<T, kLines, kAcross> L;
  static constexpr int kVec = L::kVec, kPieces = kLines * 8 / kThreads, kK = kLineBytes / sizeof(T);
  static_assert(!kPaired || kThreads / 8 <= 64, "what is loaded at once is of one of the two");
  unsigned at[kPieces];
  unsigned long long base, second, step;
  int left, blocks, part;  // left: k's to the operand's end (2^30: or more)
  unsigned id, further, lds;
  bool live;

  template <typename RunOf>
  __device__ __forceinline__ void Start(const Share &share, const RunOf &run_of, unsigned tiles, int parts, long long stride) {
    step = kAcross ? (unsigned long long)kK * stride * sizeof(T) : kLineBytes;
    further = share.of;
    id = share.first - share.of;
    part = parts - 1;
    Next(run_of, tiles, parts, stride);
  }
  template <typename RunOf>
  __device__ __forceinline__ void Next(const RunOf &run_of, unsigned tiles, int parts, long long stride) {
    Run run;
    do {
      if (++part == parts) {
        part = 0;
        id += further;
      }
      live = id < tiles;
      if (!live) {  // what is asked for from here on is from nowhere
        base = second = 0;
        left = 1 << 30;
        blocks = 0;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) at[p] = kNowhere;
        return;
      }
      run = run_of(id, part);
    } while (run.blocks <= 0);
    base = Uniform(reinterpret_cast<unsigned long long>(run.base));
    second = Uniform(reinterpret_cast<unsigned long long>(run.second));
    // (a load may read a scalar register that a vector instruction wrote, as Uniform does, five instructions later at the earliest; the compiler, which sees to
    // that elsewhere, does not know what LoadToLds is)
    asm volatile("s_nop 4" : "+s"(base), "+s"(second));
    left = (int)min(run.left, 1ll << 30);
    blocks = run.blocks;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int q = p * kThreads + threadIdx.x, line = q / L::kRowChunks, chunk = q % L::kRowChunks ^ L::Swap(line);
      const bool held = kAcross ? chunk * kVec < run.lines : RowOf<kPaired>(line) < run.lines;
      at[p] = held ? ((unsigned)RowOf<kPaired>(line) * (unsigned)stride + chunk * kVec) * (unsigned)sizeof(T) : kNowhere;
    }
  }
  // The next block goes to `to`: its loads one by one (Piece), then Done.  (Where no block is left they are from nowhere.)
  template <typename RunOf>
  __device__ __forceinline__ void Prepare(unsigned to, const RunOf &run_of, unsigned tiles, int parts, long long stride) {
    if (blocks == 0 && live) Next(run_of, tiles, parts, stride);
    if (left < kK) {  // the operand's end, and that of the run
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int q = p * kThreads + threadIdx.x, line = q / L::kRowChunks, chunk = q % L::kRowChunks ^ L::Swap(line);
        if ((kAcross ? line : chunk * kVec) >= left) at[p] = kNowhere;
      }
    }
    lds = to + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
  }
  template <int p>
  __device__ __forceinline__ void Piece() const {
    LoadToLds<p * kThreads * 16>(kPaired && (p * kThreads / 8 & 64) ? second : base, at[p], lds);
  }
  __device__ __forceinline__ void Done() {
    if (!live) return;
    base += step;
    second += step;
    left -= kK;
    --blocks;
  }
  template <typename RunOf, int... p>
  __device__ __forceinline__ void Issue(unsigned to, const RunOf &run_of, unsigned tiles, int parts, long long stride, std::integer_sequence<int, p...>) {
    Prepare(to, run_of, tiles, parts, stride);
    (Piece<p>(), ...);
    Done();
  }
  template <typename RunOf>
  __device__ __forceinline__ void Issue(unsigned to, const RunOf &run_of, unsigned tiles, int parts, long long stride) {
    Issue(to, run_of, tiles, parts, stride, std::make_integer_sequence<int, kPieces>());
  }
};

// An operand's block through registers, whatever its alignment.  (Lines beyond the operand along k: the last one again, whose results are not stored; k's
// beyond it are 0.)
template <typename T, int kLines, int kThreads, bool kAcross, bool kPaired>
struct Stage {
  typedef Layout<T, kLines, kAcross> L;
  static constexpr int kVec = L::kVec, kPieces = kLines * 8 / kThreads, kK = kLineBytes / sizeof(T);
  Chunk<T> piece[kPieces];

  __device__ __forceinline__ void Load(const Run &run, long long n, long long stride) {
    const long long left = run.left - n * kK, skip = n * kK * (kAcross ? stride : 1);
    const bool whole = left >= kK && (!kAcross || run.lines >= kLines);
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int q = p * kThreads + threadIdx.x, line = q / L::kRowChunks, chunk = q % L::kRowChunks ^ L::Swap(line);
      const T *base = static_cast<const T *>(kPaired && (p * kThreads / 8 & 64) ? run.second : run.base) + skip;
      const T *from = base + (kAcross ? line : min((long long)RowOf<kPaired>(line), run.lines - 1)) * stride + chunk * kVec;
      if (whole) {
        piece[p] = __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const Pack<T, kVec> *>(from));
      } else {
        const long long held = !kAcross ? left - chunk * kVec : line < left ? run.lines - chunk * kVec : 0;
#pragma unroll
        for (int c = 0; c < kVec; ++c) piece[p].v[c] = c < held ? from[c] : T(0);
      }
    }
  }
  __device__ __forceinline__ void Store(LdsByte *block) const {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) *(LdsI4 *)(block + (p * kThreads + threadIdx.x) * 16) = __builtin_bit_cast(I4, piece[p]);
  }
};

// What a wave sums: fragments of 16 rows by 16 columns; a lane holds row lane % 16, columns 4 (lane / 16) + 0 .. 3 of each.
template <int kFragsI>
struct Tile {
  static constexpr int kFragsJ = kWaveJ / 16;
  F4 acc[kFragsI][kFragsJ];
  __device__ __forceinline__ void Clear() {
#pragma unroll
    for (int i = 0; i < kFragsI; ++i)
#pragma unroll
      for (int j = 0; j < kFragsJ; ++j) acc[i][j] = F4{0, 0, 0, 0};
  }
  // Both halves of a block, in 16 steps of kFragsI products; between(step) after each.  What is read for a product is asked for kAhead steps ahead, and
  // steps stay as they are written: left alone the compiler reads a chunk, waits and multiplies, with as few registers as that takes.
  static constexpr int kSteps = 2 * kFragsJ, kAhead = 4;
  template <typename T, typename LayoutA, typename LayoutB, typename Between>
  __device__ __forceinline__ void Add(const LdsByte *a, const LdsByte *b, int wave_i, int wave_j, const Between &between) {
    Chunk<T> x[2][kFragsI], y[2][kFragsJ];
    const auto read_x = [&](int half, int i) { x[half][i] = LayoutA::Read(a, wave_i * kFragsI * 16 + i * 16, half); };
    const auto read_y = [&](int half, int j) { y[half][j] = LayoutB::Read(b, wave_j * kWaveJ + j * 16, half); };
#pragma unroll
    for (int i = 0; i < kFragsI; ++i) read_x(0, i);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) read_y(0, j);
    __builtin_amdgcn_sched_barrier(0);
    ForEach([&](auto step) {
      constexpr int half = step.value / kFragsJ, j = step.value % kFragsJ, soon = j + kAhead - kFragsJ;  // soon: of the next half
      if constexpr (soon < 0) {
        read_y(half, j + kAhead);
      } else if constexpr (half == 0) {
        read_y(1, soon);
        if constexpr (soon < kFragsI) read_x(1, soon);
      }
#pragma unroll
      for (int i = 0; i < kFragsI; ++i) acc[i][j] = Product(y[half][j], x[half][i], acc[i][j]);
      between(step);
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, kSteps>());
  }
  template <typename Fn, int... step>
  static __device__ __forceinline__ void ForEach(const Fn &fn, std::integer_sequence<int, step...>) {
    (fn(std::integral_constant<int, step>()), ...);
  }
};

// The blocks of a workgroup's tiles, one after the other.  kDirect: while one is multiplied, the next ones are on their way as far as the LDS holds them,
// those of the tiles that follow too while a tile's results are written.
//   run_a(id, part), run_b: the runs of a tile, `parts` of them;  add(a, b);  end(id)
template <bool kDirect, typename StreamA, typename StreamB, typename StageA, typename StageB, typename S, typename RunA, typename RunB, typename AddFn, typename EndFn>
__device__ __forceinline__ void RunTiles(LdsByte *lds, const Share &share, unsigned tiles, int parts, long long stride_a, long long stride_b, const RunA &run_a, const RunB &run_b,
                                         const AddFn &add, const EndFn &end) {
  constexpr int kA = S::kI * kLineBytes, kB = S::kJ * kLineBytes;
  if constexpr (kDirect) {
    constexpr int kAheadA = S::kBlocksA - 1, kAheadB = S::kBlocksB - 1;
    static_assert(kAheadB == kAheadA || kAheadB == kAheadA + 1, "the order of loads that follows");
    // Loads that may be on their way when a block is multiplied: those issued after its own (a block's time issues A's, then B's, of blocks further on).
    constexpr int kLater = (kAheadA - 1) * (StreamA::kPieces + StreamB::kPieces) + (kAheadB - kAheadA) * StreamB::kPieces;
    const unsigned first = __builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)lds), first_b = first + S::kBlocksA * kA;
    StreamA a;
    StreamB b;
    a.Start(share, run_a, tiles, parts, stride_a);
    b.Start(share, run_b, tiles, parts, stride_b);
    if constexpr (kAheadB > kAheadA) b.Issue(first_b, run_b, tiles, parts, stride_b);
#pragma unroll
    for (int n = 0; n < kAheadA; ++n) {
      a.Issue(first + n * kA, run_a, tiles, parts, stride_a);
      b.Issue(first_b + (n + kAheadB - kAheadA) * kB, run_b, tiles, parts, stride_b);
    }
    unsigned at_a = first, at_b = first_b, to_a = first + kAheadA * kA, to_b = first_b + kAheadB * kB;
    const auto next_a = [&](unsigned at) { return at == first + kAheadA * kA ? first : at + kA; };
    const auto next_b = [&](unsigned at) { return at == first_b + kAheadB * kB ? first_b : at + kB; };
    bool landed = false;  // whether all loads have arrived
    for (unsigned id = share.first; id < tiles; id += share.of) {
      for (int part = 0; part < parts; ++part) {
        for (int n = run_b(id, part).blocks; n > 0; --n) {
          if (landed) Meet();
          else WaitAndMeet<kLater>();
          // (the block is there, and what follows goes where the one before was, which has been read)
          landed = false;
          a.Prepare(to_a, run_a, tiles, parts, stride_a);
          b.Prepare(to_b, run_b, tiles, parts, stride_b);
          // Loads one by one between the products: all at once they fill the queue of the memory pipeline, which takes 16 cycles for each, and
          // the waves wait to issue them while nothing is multiplied.
          add((const LdsByte *)(uintptr_t)at_a, (const LdsByte *)(uintptr_t)at_b, [&](auto step) {
            constexpr int kLoads = StreamA::kPieces + StreamB::kPieces, kGap = Tile<1>::kSteps / kLoads, p = step.value / kGap;
            static_assert(kGap >= 1, "a load after every step at most");
            if constexpr (step.value % kGap == 0 && p < StreamA::kPieces) a.template Piece<p>();
            else if constexpr (step.value % kGap == 0 && p < kLoads) b.template Piece<p - StreamA::kPieces>();
          });
          a.Done();
          b.Done();
          at_a = next_a(at_a);
          at_b = next_b(at_b);
          to_a = next_a(to_a);
          to_b = next_b(to_b);
        }
      }
      // (before the tile's results are stored: a wait for loads issued before them would be one for the stores as well)
      WaitForLoads();
      landed = true;
      end(id);
    }
  } else {
    LdsByte *const to_b = lds + kA;
    for (unsigned id = share.first; id < tiles; id += share.of) {
      for (int part = 0; part < parts; ++part) {
        const Run of_a = run_a(id, part), of_b = run_b(id, part);
        StageA a;
        StageB b;
        if (of_b.blocks > 0) a.Load(of_a, 0, stride_a), b.Load(of_b, 0, stride_b);
        for (int n = 0; n < of_b.blocks; ++n) {
          __syncthreads();  // (the block before has been read)
          a.Store(lds);
          b.Store(to_b);
          __syncthreads();
          if (n + 1 < of_b.blocks) a.Load(of_a, n + 1, stride_a), b.Load(of_b, n + 1, stride_b);
          add(lds, to_b, [](auto) {});
        }
      }
      end(id);
    }
  }
}

// Workgroups that follow each other are on different XCDs: each XCD (its L2) gets tiles that lie together, eight rows of them by
// as many columns as there are.
__device__ __forceinline__ unsigned PlaceOfTile(unsigned id, unsigned all) {
  const unsigned x = id % 8, each = all / 8, rest = all % 8;
  return x * each + min(x, rest) + id / 8;
}
__device__ __forceinline__ void PlaceInGroup(unsigned tile, unsigned tile_rows, unsigned tile_columns, unsigned *i, unsigned *j) {
  const unsigned group = tile / (8 * tile_columns), first = group * 8, rows = min(tile_rows - first, 8u);
  const unsigned in = tile - group * 8 * tile_columns;
  *i = first + in % rows;
  *j = in / rows;
}

// N elements of a row from column `at` on, of `columns`.
template <typename T, int N>
__device__ __forceinline__ void StoreSome(T *row, long long at, long long columns, const Pack<T, N> &v) {
  if (at + N <= columns) {
    *reinterpret_cast<Pack<T, N> *>(row + at) = v;
  } else {
#pragma unroll
    for (int r = 0; r < N; ++r)
      if (at + r < columns) row[at + r] = v.v[r];
  }
}

// A lane's four values of each of four fragments that follow each other along a row: 64 columns from `at` on, between the four lanes of the row.  Elements of 16 and 8
// bits: the four lanes first exchange what they have of two fragments, so that each has eight columns side by side, 64 (32) bytes of the row
// between them in one store (100,003 x 64 x 256 kept as it is: 61 us with stores of four columns a lane, 46 so).
template <typename T>
__device__ __forceinline__ void StoreColumns(T *row, long long at, long long columns, const Pack<T, 4> (&v)[4]) {
  const int quarter = (threadIdx.x & 63) / 16;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) StoreSome(row, at + j * 16 + quarter * 4, columns, v[j]);
  } else {
    struct Words {
      unsigned w[sizeof(T)];
    };
    struct Both {
      Words low, high;
    };
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      // lanes' quarters 0 1 2 3 of the fragments a and b:  a0 a1 a2 a3, b0 b1 b2 b3  ->  a0 a1 b0 b1, a2 a3 b2 b3  ->  a0 a2 b0 b2, a1 a3 b1 b3
      Both p = {__builtin_bit_cast(Words, v[j]), __builtin_bit_cast(Words, v[j + 1])};
#pragma unroll
      for (int w = 0; w < (int)sizeof(T); ++w) {
        const auto halves = __builtin_amdgcn_permlane32_swap(p.low.w[w], p.high.w[w], false, false);
        const auto quarters = __builtin_amdgcn_permlane16_swap(halves[0], halves[1], false, false);
        p.low.w[w] = quarters[0];
        p.high.w[w] = quarters[1];
      }
      StoreSome(row, at + j * 16 + quarter * 8, columns, __builtin_bit_cast(Pack<T, 8>, p));
    }
  }
}

template <typename T>
__device__ __forceinline__ void StoreRounded(T *row, long long at, long long columns, const F4 *v) {
  Pack<T, 4> rounded[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) rounded[j].v[r] = Round<T>(v[j][r]);
  StoreColumns(row, at, columns, rounded);
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
  // the k's of a tile shared out
  int splits;
  long long split_blocks;
  float *partial;  // [splits][rows][groups of 64 hidden columns][64 of the gate, 64 of up]
};

// What a lane holds of four values in each of four fragments along a row: 16 of a group of 64, the other lanes of its
// row the rest.
template <typename T>
__device__ __forceinline__ void Keep(void *kept, float *scales, long long stride, long long row, int at, int hidden, const F4 *v) {
  if (scales == nullptr) {
    StoreRounded(static_cast<T *>(kept) + row * stride, at, hidden, v);
    return;
  }
  float most = 0.0f;  // (columns beyond the layer hold 0, or what the last one holds)
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) most = MostOf(most, v[j][r]);
  most = MostOf(most, __shfl_xor(most, 16));
  most = MostOf(most, __shfl_xor(most, 32));
  const float scale = ScaleOf(most);
  if ((threadIdx.x & 63) < 16) scales[row * ((hidden + kScaleGroup - 1) / kScaleGroup) + at / kScaleGroup] = scale;
  Pack<signed char, 4> codes[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float four[4] = {v[j][0], v[j][1], v[j][2], v[j][3]};
    codes[j] = CodesOf(four, scale);
  }
  StoreColumns(static_cast<signed char *>(kept) + row * stride, at, hidden, codes);
}

static_assert(kWaveJ == 2 * kScaleGroup, "a wave holds whole groups");

// A tile's columns are the gate's and up's of the same hidden ones: 64 of the gate and 64 of up for each wave, so that a lane ends with both of an element.
// The matrix instructions and the power that they take bound large layers: 8192 x 4096 x 16384 bf16 in 1662 us, 1.32 PFLOP/s (a library's plain product of that
// many operations 1.42), at 1.6 to 1.8 GHz, with the matrix units at work 60 to 66 % of the cycles; instructions of 32 x 32 x 16 took no less time and
// lowered the clock further.  Narrow ones are bound by what ends a tile: 100,003 x 64 x 256 bf16 25 us (0.064 GB, 2.6 TB/s), keeping both in 8 bits 45.
template <typename T, int kAct, typename S, bool kDirect>
__global__ void __launch_bounds__(S::kThreads) __attribute__((amdgpu_waves_per_eu(S::kWavesEach, S::kWavesEach))) k_gated(const Forward a, unsigned tiles, unsigned tile_rows, unsigned tile_columns) {
  __shared__ __align__(16) unsigned char s_blocks[kDirect ? S::kLdsBytes : (S::kI + S::kJ) * kLineBytes];
  constexpr int kK = kLineBytes / sizeof(T), kHidden = S::kJ / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wave_i = wave % (S::kI / S::kWaveI), wave_j = wave / (S::kI / S::kWaveI);
  struct At {
    long long i0, split, first;
    int h0;
  };
  const auto at_of = [&](unsigned id) {
    At at;
    const unsigned each = tile_rows * tile_columns, place = PlaceOfTile(id, tiles), split = a.splits == 1 ? 0 : place / each;
    unsigned i, j;
    PlaceInGroup(place - split * each, tile_rows, tile_columns, &i, &j);
    at.i0 = (long long)i * S::kI;
    at.h0 = j * kHidden;
    at.split = split;
    at.first = split * a.split_blocks;
    return at;
  };
  const auto blocks_of = [&](const At &at) { return (int)min(a.split_blocks, (a.dim + kK - 1) / kK - at.first); };
  const auto run_x = [&](unsigned id, int) {
    const At at = at_of(id);
    const T *x = static_cast<const T *>(a.x) + at.i0 * a.x_stride + at.first * kK;
    return Run{x, x, a.rows - at.i0, a.dim - at.first * kK, blocks_of(at)};
  };
  const auto run_w = [&](unsigned id, int) {
    const At at = at_of(id);
    const long long from = at.h0 * a.w_stride + at.first * kK;
    return Run{static_cast<const T *>(a.w_gate) + from, static_cast<const T *>(a.w_up) + from, a.hidden - at.h0, a.dim - at.first * kK, blocks_of(at)};
  };
  Tile<S::kWaveI / 16> t;
  t.Clear();
  const auto add = [&](const LdsByte *x, const LdsByte *w, const auto &between) {
    t.template Add<T, Layout<T, S::kI, false>, Layout<T, S::kJ, false>>(x, w, wave_i, wave_j, between);
  };
  RunTiles<kDirect, Stream<T, S::kI, S::kThreads, false, false>, Stream<T, S::kJ, S::kThreads, false, true>, Stage<T, S::kI, S::kThreads, false, false>,
           Stage<T, S::kJ, S::kThreads, false, true>, S>((LdsByte *)s_blocks, Share{blockIdx.x, gridDim.x}, tiles, 1, a.x_stride, a.w_stride, run_x, run_w, add, [&](unsigned id) {
    const At at = at_of(id);
    const int h = at.h0 + wave_j * (kWaveJ / 2);
#pragma unroll
    for (int i = 0; i < S::kWaveI / 16; ++i) {
      const long long row = at.i0 + wave_i * S::kWaveI + i * 16 + lane % 16;
      if (row >= a.rows || h >= a.hidden) continue;  // (all four lanes of a row)
      if (a.splits > 1) {
        float *to = a.partial + ((at.split * a.rows + row) * ((a.hidden + 63) / 64) + h / 64) * kWaveJ + lane / 16 * 4;
#pragma unroll
        for (int j = 0; j < kWaveJ / 16; ++j) *reinterpret_cast<F4 *>(to + j * 16) = t.acc[i][j];
        continue;
      }
      F4 out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) out[j][r] = Act<kAct>(t.acc[i][j][r]) * t.acc[i][j + 4][r];
      StoreRounded(static_cast<T *>(a.out) + row * a.out_stride, h, a.hidden, out);
      if (a.gate != nullptr) {
        Keep<T>(a.gate, a.gate_scales, a.kept_stride, row, h, a.hidden, t.acc[i]);
        Keep<T>(a.up, a.up_scales, a.kept_stride, row, h, a.hidden, t.acc[i] + 4);
      }
    }
    t.Clear();
  });
}

constexpr int kThreads = 256;  // of the kernels that go element by element

// What was shared out: a wave sums 64 hidden columns of a row, in order, and ends as a tile does.
template <typename T, int kAct>
__global__ void __launch_bounds__(kThreads) k_gated_join(const Forward a, long long items) {
  const int lane = threadIdx.x & 63, groups = (a.hidden + 63) / 64;
  const long long step = a.rows * groups * kWaveJ;
  for (long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); item < items; item += (long long)gridDim.x * 4) {
    const long long row = item / groups;
    const int group = (int)(item - row * groups), h = group * 64 + lane;
    const float *from = a.partial + item * kWaveJ + lane;
    float g = from[0], u = from[64];
    for (int split = 1; split < a.splits; ++split) {
      g += from[split * step];
      u += from[split * step + 64];
    }
    const bool there = h < a.hidden;
    if (there) static_cast<T *>(a.out)[row * a.out_stride + h] = Round<T>(Act<kAct>(g) * u);
    if (a.gate == nullptr) continue;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float v = which == 0 ? g : u;
      void *kept = which == 0 ? a.gate : a.up;
      float *scales = which == 0 ? a.gate_scales : a.up_scales;
      if (scales == nullptr) {
        if (there) static_cast<T *>(kept)[row * a.kept_stride + h] = Round<T>(v);
        continue;
      }
      float most = there ? fabsf(v) : 0.0f;
#pragma unroll
      for (int by = 32; by > 0; by /= 2) most = MostOf(most, __shfl_xor(most, by));
      const float scale = ScaleOf(most);
      if (lane == 0) scales[row * groups + group] = scale;
      const float one[1] = {v};
      if (there) static_cast<signed char *>(kept)[row * a.kept_stride + h] = CodesOf(one, scale).v[0];
    }
  }
}

// Few rows (up to 16): 16 hidden columns a workgroup, whose eight waves share out the k's.  The weights are read once, from memory into the
// registers that the products take them from: a lane's chunk is 16 bytes of a weight row, four steps of 64 bytes a row at once.
// kApart: rows that begin anywhere.  Every eighth of them begins alike within 16 bytes, and the workgroup takes sixteen of those; behind as many k's as
// the row's first 16 bytes hold its chunks are aligned.  (In which order a sum is formed, and so its last bits, then depend on where the weights lie.)  Reading the weights bounds it: 1 x 4096 x 16384 bf16 48 us, 5.6 TB/s.
constexpr int kFewWaves = 8;
template <typename T, int kAct, bool kApart>
__global__ void __launch_bounds__(64 * kFewWaves) k_gated_few(const Forward a) {
  constexpr int kVec = 16 / sizeof(T), kStep = 4 * kVec, kUnroll = 4, kEach = kApart ? 8 : 1;  // kEach: rows from one to the next
  __shared__ float s_sums[kFewWaves][2][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane / 16;
  const int h0 = kApart ? blockIdx.x / 8 * 128 + blockIdx.x % 8 : blockIdx.x * 16;
  if (h0 >= a.hidden) return;
  const long long h = h0 + lane % 16 * kEach < a.hidden ? h0 + lane % 16 * kEach : h0, i = min(lane % 16ll, a.rows - 1);
  int head = 0;
  if (kApart) head = min((int)((16 - reinterpret_cast<uintptr_t>(static_cast<const T *>(a.w_gate) + h0 * a.w_stride) % 16) % 16 / sizeof(T)), a.dim);
  const int at = head + quarter * kVec;
  const T *gate = static_cast<const T *>(a.w_gate) + h * a.w_stride + at, *up = static_cast<const T *>(a.w_up) + h * a.w_stride + at;
  const T *x = static_cast<const T *>(a.x) + i * a.x_stride + at;
  F4 g = {0, 0, 0, 0}, u = {0, 0, 0, 0};
  const int steps = (a.dim - head + kStep - 1) / kStep, groups = (a.dim - head) / kStep / kUnroll;
  const auto whole = [&](const T *from) { return __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const Pack<T, kVec> *>(from)); };
  for (int group = wave; group < groups; group += kFewWaves) {
    Chunk<T> gs[kUnroll], us[kUnroll], xs[kUnroll];
#pragma unroll
    for (int n = 0; n < kUnroll; ++n) {
      const int k = (group * kUnroll + n) * kStep;
      gs[n] = whole(gate + k);
      us[n] = whole(up + k);
      xs[n] = whole(x + k);
    }
#pragma unroll
    for (int n = 0; n < kUnroll; ++n) {
      g = Product(gs[n], xs[n], g);
      u = Product(us[n], xs[n], u);
    }
  }
  // what is left, a step a wave: up to four at the end, and the k's before `head`
  static_assert(kUnroll < kFewWaves, "a wave for each step that is left, and one for the head");
  const bool first = kApart && wave == kFewWaves - 1;
  const int step = groups * kUnroll + wave;
  if (first ? head > 0 : step < steps) {
    const int k = first ? -at : step * kStep, held = !first ? a.dim - at - k : quarter == 0 ? head : 0;
    const auto part = [&](const T *from) {
      Chunk<T> c;
#pragma unroll
      for (int e = 0; e < kVec; ++e) c.v[e] = e < held ? from[e] : T(0);
      return c;
    };
    const Chunk<T> xs = part(x + k);
    g = Product(part(gate + k), xs, g);
    u = Product(part(up + k), xs, u);
  }
  *reinterpret_cast<F4 *>(&s_sums[wave][0][lane * 4]) = g;
  *reinterpret_cast<F4 *>(&s_sums[wave][1][lane * 4]) = u;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int in = threadIdx.x, of = in / 4, row = of % 16, column = h0 + (of / 16 * 4 + in % 4) * kEach;  // of: the lane that held it
  if (row >= a.rows || column >= a.hidden) return;
  float gv = 0.0f, uv = 0.0f;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) {
    gv += s_sums[w][0][in];
    uv += s_sums[w][1][in];
  }
  static_cast<T *>(a.out)[row * a.out_stride + column] = Round<T>(Act<kAct>(gv) * uv);
  if (a.gate != nullptr) {
    static_cast<T *>(a.gate)[row * a.kept_stride + column] = Round<T>(gv);
    static_cast<T *>(a.up)[row * a.kept_stride + column] = Round<T>(uv);
  }
}

// Up to three matrices of rows that begin anywhere, to rows that begin at multiples of 64 elements, 0 behind each row's end.  (x and both weights of 1003 x 771 x 2055 fp16,
// 16 MB read and written: 8 us; 290 MB in rows of 3033 57, 5.1 TB/s.)
struct Padded {
  const void *from[3];
  void *to[3];
  long long rows[3], from_stride[3];
  int width;
  long long to_stride, blocks;  // blocks: of kThreads vectors
};
template <typename T>
__device__ __forceinline__ void PadRows(const Share &share, const Padded &a) {
  constexpr int kVec = 8;
  const unsigned vectors = (unsigned)(a.to_stride / kVec);
  for (long long block = share.first; block < a.blocks; block += share.of) {
    const long long first = block * kThreads, row0 = first / vectors;
    const unsigned in = (unsigned)(first - row0 * vectors) + threadIdx.x, more = in / vectors;
    long long row = row0 + more;
    // (no index that is not a constant: such a one puts the arguments into scratch memory)
    const void *of = a.from[0];
    void *to = a.to[0];
    long long stride = a.from_stride[0];
    if (row >= a.rows[0]) row -= a.rows[0], of = a.from[1], to = a.to[1], stride = a.from_stride[1];
    if (to == a.to[1] && row >= a.rows[1]) row -= a.rows[1], of = a.from[2], to = a.to[2], stride = a.from_stride[2];
    if (to == a.to[2] && row >= a.rows[2]) continue;
    const int at = (int)(in - more * vectors) * kVec, held = a.width - at;
    const T *from = static_cast<const T *>(of) + row * stride + at;
    Pack<T, kVec> p;
    if (held >= kVec) {
      p = *reinterpret_cast<const Pack<T, kVec> *>(from);
    } else {
#pragma unroll
      for (int c = 0; c < kVec; ++c) p.v[c] = c < held ? from[c] : T(0);
    }
    *reinterpret_cast<Pack<T, kVec> *>(static_cast<T *>(to) + row * a.to_stride + at) = p;
  }
}
template <typename T>
__global__ void __launch_bounds__(kThreads) k_pad(const Padded a) {
  PadRows<T>(Share{blockIdx.x, gridDim.x}, a);
}

// What a product's tiles are, and how many.
struct TilesOf {
  unsigned all, rows, columns;
};

// Products of the gradient.  Operands that lie across are turned on their way from the LDS to the registers, by reads made for that, so neither is copied first.  The
// matrix instructions and their power bound it as they do the layer: 4096 x 4096 x 16384 bf16, d_gate Wg + d_up Wu 840 us, 1.31 PFLOP/s, and both weights' 870, 1.26.
template <typename T, bool kAcrossA, bool kAcrossB, typename S, bool kDirect>
__device__ __forceinline__ void RunProducts(LdsByte *lds, const Share &share, const Products &p, const TilesOf &tiles) {
  constexpr int kK = kLineBytes / sizeof(T);
  const long long segment_blocks = (p.inner + kK - 1) / kK;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wave_i = wave % (S::kI / S::kWaveI), wave_j = wave / (S::kI / S::kWaveI);
  struct At {
    long long i0, one, first;
    int j0, member;
  };
  const auto at_of = [&](unsigned id) {
    At at;
    const unsigned each = tiles.rows * tiles.columns, place = PlaceOfTile(id, tiles.all), one = place / each, member = one / (unsigned)p.splits;
    unsigned i, j;
    PlaceInGroup(place - one * each, tiles.rows, tiles.columns, &i, &j);
    at.i0 = (long long)i * S::kI;
    at.j0 = j * S::kJ;
    at.one = one;
    at.member = member;
    at.first = (one - member * p.splits) * p.split_blocks;
    return at;
  };
  // A tile's blocks of k's in each segment.
  const auto run_of = [&](const At &at, int segment, const Operand &of, bool across, long long row0, long long rows) {
    const long long begin = max(at.first, segment * segment_blocks), end = min(at.first + p.split_blocks, (segment + 1) * segment_blocks);
    const long long k0 = (begin - segment * segment_blocks) * kK;
    const T *base = static_cast<const T *>(of.at[at.member + segment]) + (across ? k0 * of.stride + row0 : row0 * of.stride + k0);
    return Run{base, base, rows - row0, p.inner - k0, (int)max(end - begin, 0ll)};
  };
  const auto run_a = [&](unsigned id, int segment) {
    const At at = at_of(id);
    return run_of(at, segment, p.a, kAcrossA, at.i0, p.rows);
  };
  const auto run_b = [&](unsigned id, int segment) {
    const At at = at_of(id);
    return run_of(at, segment, p.b, kAcrossB, at.j0, p.columns);
  };
  Tile<S::kWaveI / 16> t;
  t.Clear();
  const float undo = UndoOf<T>(p);
  const auto add = [&](const LdsByte *of_a, const LdsByte *of_b, const auto &between) {
    t.template Add<T, Layout<T, S::kI, kAcrossA>, Layout<T, S::kJ, kAcrossB>>(of_a, of_b, wave_i, wave_j, between);
  };
  RunTiles<kDirect, Stream<T, S::kI, S::kThreads, kAcrossA, false>, Stream<T, S::kJ, S::kThreads, kAcrossB, false>, Stage<T, S::kI, S::kThreads, kAcrossA, false>,
           Stage<T, S::kJ, S::kThreads, kAcrossB, false>, S>(lds, share, tiles.all, p.segments, p.a.stride, p.b.stride, run_a, run_b, add, [&](unsigned id) {
    const At at = at_of(id);
#pragma unroll
    for (int i = 0; i < S::kWaveI / 16; ++i) {
      const long long row = at.i0 + wave_i * S::kWaveI + i * 16 + lane % 16;
      if (row >= p.rows) continue;
#pragma unroll
      for (int j = 0; j < kWaveJ / 16; j += 4) {
        const int column = at.j0 + wave_j * kWaveJ + j * 16;
        if (p.splits > 1) {
          StoreRounded(p.partial + (at.one * p.rows + row) * p.columns, column, p.columns, &t.acc[i][j]);
          continue;
        }
        if constexpr (std::is_same_v<T, _Float16>) {
#pragma unroll
          for (int f = 0; f < 4; ++f) t.acc[i][j + f] *= undo;
        }
        StoreRounded(static_cast<T *>(p.c[at.member]) + row * p.c_stride, column, p.columns, &t.acc[i][j]);
      }
    }
    t.Clear();
  });
}

template <typename T, bool kAcrossA, bool kAcrossB, typename S, bool kDirect>
__global__ void __launch_bounds__(S::kThreads) __attribute__((amdgpu_waves_per_eu(S::kWavesEach, S::kWavesEach))) k_products(const Products p, const TilesOf tiles) {
  __shared__ __align__(16) unsigned char s_blocks[kDirect ? S::kLdsBytes : (S::kI + S::kJ) * kLineBytes];
  RunProducts<T, kAcrossA, kAcrossB, S, kDirect>((LdsByte *)s_blocks, Share{blockIdx.x, gridDim.x}, p, tiles);
}

// grad_x and the weights' gradients side by side, `x_groups` workgroups for the first, where all tiles of both have a place on the chip at once: a layer that
// small waits for its loads, not for what it shares with the other (bf16, forward and gradient, one after the other and so: 1003 x 771 x 2055 93 and 71 us,
// 2000 x 300 x 500 53 and 41, 3000 x 1000 x 1000 88 and 68).
template <typename T>
__global__ void __launch_bounds__(SmallTile::kThreads) __attribute__((amdgpu_waves_per_eu(SmallTile::kWavesEach, SmallTile::kWavesEach)))
k_both_products(const Products x, const TilesOf x_tiles, unsigned x_groups, const Products w, const TilesOf w_tiles) {
  __shared__ __align__(16) unsigned char s_blocks[SmallTile::kLdsBytes];
  if (blockIdx.x < x_groups) RunProducts<T, false, true, SmallTile, true>((LdsByte *)s_blocks, Share{blockIdx.x, x_groups}, x, x_tiles);
  else RunProducts<T, true, true, SmallTile, true>((LdsByte *)s_blocks, Share{blockIdx.x - x_groups, gridDim.x - x_groups}, w, w_tiles);
}

// The sums of what was shared out, in an order that depends on the sizes alone: four elements side by side a thread, or many shares by kShares threads,
// each with every kShares-th of them.  (Many shares mean few elements: 63 of 2 x 256 x 64 by a thread each take 17.7 us, by eight 5.)
template <typename T, int kShares>
__device__ __forceinline__ void JoinProducts(const Share &share_of, const Products &p) {
  constexpr int kVec = kShares == 1 ? 4 : 1, kElements = kThreads / kShares * kVec;
  __shared__ float s_sums[kShares][kShares == 1 ? 1 : kElements];
  const long long each = p.rows * p.columns, step = (long long)share_of.of * kElements;
  const float undo = UndoOf<T>(p);
  const int in = threadIdx.x % (kThreads / kShares) * kVec, share = threadIdx.x / (kThreads / kShares);
  for (int member = 0; member < p.batch; ++member) {
    T *c = static_cast<T *>(p.c[member]);
    for (long long first = (long long)share_of.first * kElements; first < each; first += step) {
      const long long at = first + in;
      const float *from = p.partial + (long long)member * p.splits * each + at;
      const int held = (int)max(0ll, min(each - at, (long long)kVec));
      float sum[kVec] = {};
      for (int s = share; s < p.splits; s += kShares) {
        if (held == kVec) {
          const Pack<float, kVec> v = *reinterpret_cast<const Pack<float, kVec> *>(from + s * each);
#pragma unroll
          for (int e = 0; e < kVec; ++e) sum[e] += v.v[e];
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e) sum[e] += e < held ? from[s * each + e] : 0.0f;
        }
      }
      if constexpr (kShares > 1) {
        s_sums[share][in] = sum[0];
        __syncthreads();
        sum[0] = s_sums[0][in];
#pragma unroll
        for (int s = 1; s < kShares; ++s) sum[0] += s_sums[s][in];
        __syncthreads();
      }
      if (held == 0 || share != 0) continue;
      if constexpr (std::is_same_v<T, _Float16>) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum[e] *= undo;
      }
      const long long row = each < (1ll << 32) ? (long long)((unsigned)at / (unsigned)p.columns) : at / p.columns;
      const int column = (int)(at - row * p.columns);
      if (column + kVec <= p.columns) {
        Pack<T, kVec> rounded;
#pragma unroll
        for (int e = 0; e < kVec; ++e) rounded.v[e] = Round<T>(sum[e]);
        *reinterpret_cast<Pack<T, kVec> *>(c + row * p.c_stride + column) = rounded;
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          if (e >= held) break;
          const int over = (column + e) / p.columns;  // rows further on
          c[(row + over) * p.c_stride + column + e - over * p.columns] = Round<T>(sum[e]);
        }
      }
    }
  }
}

constexpr int kManyShares = 16;

// Of one product, or of two: `groups` workgroups for the first.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_products_join(const Products first, unsigned groups, const Products second) {
  const auto join = [](const Share &share, const Products &p) {
    if (p.splits >= kManyShares) JoinProducts<T, 8>(share, p);
    else JoinProducts<T, 1>(share, p);
  };
  if (blockIdx.x < groups) join(Share{blockIdx.x, groups}, first);
  else join(Share{blockIdx.x - groups, gridDim.x - groups}, second);
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
  float *range;  // float16: [1 + workgroup] the greatest finite magnitude of what it formed; [0] what undoes the factor
};

constexpr int kSlopeVec = 8;

// The greatest of a workgroup's values, to all of its threads.
__device__ __forceinline__ float MostOfGroup(float most) {
  __shared__ float s_most[kThreads / 64];
#pragma unroll
  for (int by = 32; by > 0; by /= 2) most = fmaxf(most, __shfl_xor(most, by));
  if ((threadIdx.x & 63) == 0) s_most[threadIdx.x >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) most = fmaxf(most, s_most[w]);
  return most;
}

// The power of two that factors of which `most` is the greatest are taken times in float16 (as far as its reciprocal is a normal number).
__device__ __forceinline__ float FactorFor(float most) {
  if (most == 0.0f || (most >= 1.0f && most < 65504.0f)) return 1.0f;
  return ldexpf(1.0f, min(14 - ilogbf(most), 126));
}

// d_gate and d_up; 0 in the columns from the layer's end to the next row.  A thread has kSlopeVec columns of a row (d_stride is a multiple of 64).
// Both are rounded to the layer's type, which the matrix instructions of the products they enter take: half a step of each term, on top of the half
// step that gate and up were kept at, which is what sets the gradients of 16-bit layers off (rms 3e-3 of their size in bf16, where products of float32
// operands, rounded at the end, are off by 1.7e-3).  A second part for what rounding leaves would double the products' work.
// Memory bounds it: 4096 x 16384 bf16, 0.67 GB, 121 us, 5.6 TB/s; from 8 bits, 100,003 x 256, 0.21 GB, 39 us.
// Workgroups from `groups` on copy to aligned rows what the products need there.
// float16 does not hold what float32 forms of its numbers: 2^11 times 64 is infinite in it, 2^-20 times 2^-8 is 0, while the sums over them may well be numbers of
// it.  So this pass also finds the greatest (finite) magnitude, and a second one (kAgain) takes both times a power of two that brings it to 2^14 or more, undone where
// the products end, unless it lies from 1 to float16's greatest number: there what is taken as it is loses no more than 2^-25 of the greatest, as much as
// float32 sums with it would.  The second pass then ends as it has seen that.  (fp16, us, in one pass and so: 100,003 x 256 from 8 bits 37 and 46 + 5,
// 4096 x 16384 123 and 135 + 6, 1003 x 2055 9 and 11 + 4.  A pass for the magnitudes alone, before, would read all that this one reads.)
template <typename T, int kAct, bool kCodes, bool kAgain>
__global__ void __launch_bounds__(kThreads) k_slopes(const Slopes a, long long blocks, unsigned groups, const Padded pad) {
  typedef std::conditional_t<kCodes, signed char, T> Kept;
  const unsigned vectors = (unsigned)(a.d_stride / kSlopeVec);
  if (blockIdx.x >= groups) {
    PadRows<T>(Share{blockIdx.x - groups, gridDim.x - groups}, pad);
    return;
  }
  constexpr bool kRange = std::is_same_v<T, _Float16>;
  float most = 0.0f, factor = 1.0f;
  if constexpr (kAgain) {
    for (unsigned g = threadIdx.x; g < groups; g += kThreads) most = fmaxf(most, a.range[1 + g]);
    factor = FactorFor(MostOfGroup(most));
    if (blockIdx.x == 0 && threadIdx.x == 0) a.range[0] = 1.0f / factor;
    if (factor == 1.0f) return;
  }
  for (long long block = blockIdx.x; block < blocks; block += groups) {
    const long long first = block * kThreads, row0 = first / vectors;
    const unsigned in = (unsigned)(first - row0 * vectors) + threadIdx.x, more = in / vectors;
    const long long row = row0 + more;
    if (row >= a.rows) continue;
    const int at = (int)(in - more * vectors) * kSlopeVec, held = min(a.hidden - at, kSlopeVec);
    const T *grad = static_cast<const T *>(a.grad_out) + row * a.grad_out_stride + at;
    const Kept *gate = static_cast<const Kept *>(a.gate) + row * a.kept_stride + at, *up = static_cast<const Kept *>(a.up) + row * a.kept_stride + at;
    Pack<T, kSlopeVec> y;
    Pack<Kept, kSlopeVec> g, u;
    float gate_scale = 0.0f, up_scale = 0.0f;
    if (kCodes) {
      const long long group = row * (a.d_stride / kScaleGroup) + at / kScaleGroup;
      gate_scale = a.gate_scales[group];
      up_scale = a.up_scales[group];
    }
    if (held == kSlopeVec) {
      y = *reinterpret_cast<const Pack<T, kSlopeVec> *>(grad);
      g = *reinterpret_cast<const Pack<Kept, kSlopeVec> *>(gate);
      u = *reinterpret_cast<const Pack<Kept, kSlopeVec> *>(up);
    } else {
#pragma unroll
      for (int c = 0; c < kSlopeVec; ++c) {
        y.v[c] = c < held ? grad[c] : T(0);
        g.v[c] = c < held ? gate[c] : Kept(0);
        u.v[c] = c < held ? up[c] : Kept(0);
      }
    }
    Pack<T, kSlopeVec> dg, du;
#pragma unroll
    for (int c = 0; c < kSlopeVec; ++c) {
      float gv, uv;
      if constexpr (kCodes) {
        gv = Restored(g.v[c], gate_scale);
        uv = Restored(u.v[c], up_scale);
      } else {
        gv = (float)g.v[c];
        uv = (float)u.v[c];
      }
      float act, slope;
      ActAndSlope<kAct>(gv, &act, &slope);
      const bool there = c < held;
      if constexpr (kRange && !kAgain) {
        // (products of its own: the instruction that rounds those below to 16 bits multiplies as well, where nothing else needs them, and rounds once)
        float of[2] = {slope, act};
        asm("" : "+v"(of[0]), "+v"(of[1]));
        const float d[2] = {fabsf((float)y.v[c] * uv * of[0]), fabsf((float)y.v[c] * of[1])};
#pragma unroll
        for (int w = 0; w < 2; ++w) most = there && d[w] < __builtin_inff() ? fmaxf(most, d[w]) : most;
      }
      dg.v[c] = there ? Round<T>(kAgain ? (float)y.v[c] * uv * slope * factor : (float)y.v[c] * uv * slope) : T(0);
      du.v[c] = there ? Round<T>(kAgain ? (float)y.v[c] * act * factor : (float)y.v[c] * act) : T(0);
    }
    *reinterpret_cast<Pack<T, kSlopeVec> *>(static_cast<T *>(a.d_gate) + row * a.d_stride + at) = dg;
    *reinterpret_cast<Pack<T, kSlopeVec> *>(static_cast<T *>(a.d_up) + row * a.d_stride + at) = du;
  }
  if constexpr (kRange && !kAgain) {
    most = MostOfGroup(most);
    if (threadIdx.x == 0) a.range[1 + blockIdx.x] = most;
  }
}

// ------------------------------------------------------------------ launches

constexpr long long kMostGrid = 1 << 20, kCus = 256;

template <typename Fn>
void WithActivation(int activation, Fn &&fn) {
  if (activation == kSilu) fn(std::integral_constant<int, kSilu>());
  else fn(std::integral_constant<int, kGelu>());
}

// Whether an operand's chunks are aligned and whole, and its tiles within what a load's offset spans.
template <typename T>
bool IsDirect(const void *p, long long stride, long long extent) {
  const long long item = sizeof(T);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * item % 16 == 0 && extent * item % 16 == 0 && stride * item * 256 < (1ll << 31) - (1 << 20);
}

inline unsigned CheckedTiles(long long tiles) {
  if (tiles >= (1ll << 30)) throw std::runtime_error("the layer is too large");
  return (unsigned)tiles;
}

template <typename S>
TilesOf TilesFor(const Products &p) {
  const long long rows = Pieces(p.rows, S::kI), columns = Pieces(p.columns, S::kJ);
  return TilesOf{CheckedTiles(rows * columns * p.batch * p.splits), (unsigned)rows, (unsigned)columns};
}

// Workgroups for the joining of a product's shares; 0 where there are none.
inline unsigned JoinGroups(const Products &p) {
  if (p.splits <= 1) return 0;
  return (unsigned)std::min(Pieces(p.rows * p.columns, p.splits >= kManyShares ? kThreads / 8 : kThreads * 4), kMostGrid);
}

template <typename T, bool kAcrossA, bool kAcrossB>
void Launch(const Products &p, bool large, bool direct, hipStream_t stream) {
  const auto launch = [&](auto shape, auto is_direct) {
    typedef decltype(shape) S;
    const TilesOf tiles = TilesFor<S>(p);
    hipLaunchKernelGGL((k_products<T, kAcrossA, kAcrossB, S, decltype(is_direct)::value>), dim3(std::min(tiles.all, (unsigned)(kCus * S::kEach))), dim3(S::kThreads), 0, stream, p, tiles);
  };
  if (large && direct) launch(LargeTile(), std::true_type());
  else if (direct) launch(SmallTile(), std::true_type());
  else launch(SmallTile(), std::false_type());
  if (const unsigned groups = JoinGroups(p)) hipLaunchKernelGGL((k_products_join<T>), dim3(groups), dim3(kThreads), 0, stream, p, groups, p);
}

// x and the two weights in rows that begin at multiples of 64 elements, where the plan has room for that: how they get there, with the layer's pointers set to
// them.  (No blocks: nowhere.)
inline Padded PadOf(GatedLayer *l, const LayerPad &pad, bool x, bool weights, unsigned char *work) {
  if (pad.stride == 0) return Padded{};
  Padded p{{l->x, l->w_gate, l->w_up}, {work + pad.x, work + pad.w_gate, work + pad.w_up}, {x ? l->rows : 0, weights ? l->hidden : 0, weights ? l->hidden : 0},
           {l->x_stride, l->w_stride, l->w_stride}, l->dim, pad.stride, 0};
  p.blocks = Pieces((p.rows[0] + p.rows[1] + p.rows[2]) * (pad.stride / 8), kThreads);
  l->x = p.to[0];
  l->w_gate = p.to[1];
  l->w_up = p.to[2];
  l->x_stride = l->w_stride = pad.stride;
  return p;
}
inline unsigned GroupsOf(const Padded &p) { return (unsigned)std::min(p.blocks, kMostGrid); }

}  // namespace

template <typename T>
void RunGated(const GatedArgs &a, const GatedPlan &plan) {
  GatedLayer l = a.layer;
  const hipStream_t stream = static_cast<hipStream_t>(l.stream);
  unsigned char *work = static_cast<unsigned char *>(l.work);
  const bool few = plan.few && !l.gate_scales;
  const Padded pad = few ? Padded{} : PadOf(&l, plan.pad, true, true, work);
  if (pad.blocks > 0) hipLaunchKernelGGL((k_pad<T>), dim3(GroupsOf(pad)), dim3(kThreads), 0, stream, pad);
  const long long extent = pad.blocks > 0 ? plan.pad.stride : l.dim;
  const bool direct = IsDirect<T>(l.x, l.x_stride, extent) && IsDirect<T>(l.w_gate, l.w_stride, extent) && IsDirect<T>(l.w_up, l.w_stride, extent);
  const Forward f{l.x, l.w_gate, l.w_up, l.rows, l.dim, l.hidden, l.x_stride, l.w_stride, a.out, a.out_stride, l.gate, l.up, l.gate_scales,
                  l.up_scales, l.kept_stride, (int)plan.out.splits, plan.out.split_blocks, reinterpret_cast<float *>(work + plan.partial)};
  WithActivation(l.activation, [&](auto act) {
    constexpr int kAct = decltype(act)::value;
    if (few) {
      if constexpr (sizeof(T) == 2) {
        // Rows that begin at odd elements, in both weights alike: loads at less than four bytes' alignment take twice as long (bf16, 1 row of 4095 x 16383 102 us,
        // apart 61; of 4094 x 16383, whose rows lie on four bytes, 65, apart 67).
        if (l.w_stride % 2 != 0 && (reinterpret_cast<uintptr_t>(l.w_gate) - reinterpret_cast<uintptr_t>(l.w_up)) % 16 == 0) {
          hipLaunchKernelGGL((k_gated_few<T, kAct, true>), dim3((unsigned)Pieces(l.hidden, 128) * 8), dim3(64 * kFewWaves), 0, stream, f);
          return;
        }
      }
      hipLaunchKernelGGL((k_gated_few<T, kAct, false>), dim3((unsigned)Pieces(l.hidden, 16)), dim3(64 * kFewWaves), 0, stream, f);
      return;
    }
    const auto launch = [&](auto shape, auto is_direct) {
      typedef decltype(shape) S;
      const long long tile_rows = Pieces(l.rows, S::kI), tile_columns = Pieces(l.hidden, S::kJ / 2), tiles = tile_rows * tile_columns * f.splits;
      hipLaunchKernelGGL((k_gated<T, kAct, S, decltype(is_direct)::value>), dim3((unsigned)std::min(tiles, kCus * S::kEach)), dim3(S::kThreads), 0, stream, f,
                         CheckedTiles(tiles), (unsigned)tile_rows, (unsigned)tile_columns);
    };
    if (plan.out.large && direct) launch(LargeTile(), std::true_type());
    else if (direct) launch(SmallTile(), std::true_type());
    else launch(SmallTile(), std::false_type());
    if (f.splits > 1) {
      const long long items = l.rows * Pieces(l.hidden, 64);
      hipLaunchKernelGGL((k_gated_join<T, kAct>), dim3((unsigned)std::min(Pieces(items, 4), kMostGrid)), dim3(kThreads), 0, stream, f, items);
    }
  });
  HIP_OK(hipGetLastError());
}

template <typename T>
void RunGatedGrad(const GatedGradArgs &a, const GatedGradPlan &plan) {
  GatedLayer l = a.layer;
  const hipStream_t stream = static_cast<hipStream_t>(l.stream);
  unsigned char *work = static_cast<unsigned char *>(l.work);
  void *d_gate = work + plan.d_gate, *d_up = work + plan.d_up;
  constexpr bool kRange = std::is_same_v<T, _Float16>;
  float *range = kRange && l.rows > 0 ? reinterpret_cast<float *>(work + plan.range) : nullptr;
  const Padded pad = PadOf(&l, plan.pad, a.grad_w_gate != nullptr, a.grad_x != nullptr, work);
  const long long extent = pad.blocks > 0 ? plan.pad.stride : l.dim;
  if (l.rows > 0) {
    const Slopes s{a.grad_out, a.grad_out_stride, l.gate, l.up, l.gate_scales, l.up_scales, l.kept_stride, d_gate, d_up, plan.d_stride, l.rows, l.hidden, range};
    const long long blocks = Pieces(l.rows * (plan.d_stride / kSlopeVec), kThreads);
    const unsigned groups = (unsigned)(kRange ? Pieces(blocks, Pieces(blocks, kRangeGroups)) : std::min(blocks, kMostGrid));
    const auto launch = [&](auto act, auto codes, auto again, const Padded &copies) {
      hipLaunchKernelGGL((k_slopes<T, decltype(act)::value, decltype(codes)::value, decltype(again)::value>), dim3(groups + GroupsOf(copies)), dim3(kThreads), 0, stream, s,
                         blocks, groups, copies);
    };
    WithActivation(l.activation, [&](auto act) {
      if (l.gate_scales) launch(act, std::true_type(), std::false_type(), pad);
      else launch(act, std::false_type(), std::false_type(), pad);
      if constexpr (kRange) {
        if (l.gate_scales) launch(act, std::true_type(), std::true_type(), Padded{});
        else launch(act, std::false_type(), std::true_type(), Padded{});
      }
    });
  }
  const Operand d{{d_gate, d_up}, plan.d_stride};
  const bool d_direct = IsDirect<T>(d_gate, plan.d_stride, plan.d_stride);
  const Products x{d, {{l.w_gate, l.w_up}, l.w_stride}, l.rows, l.dim, l.hidden, 2, 1, {a.grad_x, nullptr}, a.grad_x_stride,
                   (int)plan.x.splits, plan.x.split_blocks, reinterpret_cast<float *>(work + plan.x_partial), range};
  const Products w{d, {{l.x, l.x}, l.x_stride}, l.hidden, l.dim, l.rows, 1, 2, {a.grad_w_gate, a.grad_w_up}, a.grad_w_stride,
                   (int)plan.w.splits, plan.w.split_blocks, reinterpret_cast<float *>(work + plan.w_partial), range};
  const bool x_direct = d_direct && IsDirect<T>(l.w_gate, l.w_stride, extent) && IsDirect<T>(l.w_up, l.w_stride, extent);
  const bool w_direct = d_direct && IsDirect<T>(l.x, l.x_stride, extent), wants_x = a.grad_x && l.rows > 0;
  if (plan.together && wants_x && a.grad_w_gate && x_direct && w_direct) {
    const TilesOf x_tiles = TilesFor<SmallTile>(x), w_tiles = TilesFor<SmallTile>(w);
    hipLaunchKernelGGL((k_both_products<T>), dim3(x_tiles.all + w_tiles.all), dim3(SmallTile::kThreads), 0, stream, x, x_tiles, x_tiles.all, w, w_tiles);
    const unsigned x_groups = JoinGroups(x), w_groups = JoinGroups(w);
    if (x_groups + w_groups > 0) hipLaunchKernelGGL((k_products_join<T>), dim3(x_groups + w_groups), dim3(kThreads), 0, stream, x, x_groups, w);
  } else {
    if (wants_x) Launch<T, false, true>(x, plan.x.large, x_direct, stream);
    if (a.grad_w_gate) Launch<T, true, true>(w, plan.w.large, w_direct, stream);
  }
  HIP_OK(hipGetLastError());
}

}  // namespace arb
#endif  // ARBORETUM_AMD_GATED_KERNELS_H_
