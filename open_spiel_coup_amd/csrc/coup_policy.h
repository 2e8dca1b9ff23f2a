// coup_policy.h -- the learner-side operators over the env's trajectories
// (include/coup_mi355x.h, "learner-side operators"): masked action sampling,
// turn-based generalised advantages, the clipped policy loss and the paired
// log-ratio preference loss, forward and gradient.
//
// A row is one decision: A <= 31 logits, its legal-action word, its action.
// A row counts where the action is legal: 0 <= action < A, the word's bit
// `action` set, bit 31 (a chance node) clear.  Rows that do not count are
// never computed on, so whatever their logits, old log probabilities and
// advantages hold cannot reach an output.  One thread works on one row, whose
// logits it keeps in registers, padded to AP (an illegal or padded action is
// -inf, which every sum below takes as 0); a block's 256 rows go through LDS.
//
// Arithmetic: logits are widened to 32 bits on load; the softmax statistics,
// the log probabilities and the gradient are 32-bit; the losses' sums over
// rows are 64-bit.  A gradient is rounded once, to the logits' type, at its
// store.  Two comparisons decide whole outputs and are repeated in 64 bits where 32-bit
// rounding could turn them: which action a uniform number falls on, and which
// side of the clip border a ratio is on.
//
// What bounds them: the bytes of the tables.  The figures at the kernels are
// of one MI355X, where a copy of 4 GiB runs at 4.65 TB/s (reads and writes)
// and one of 64 MiB, in the last-level cache, at 6.9.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "coup_mi355x.h"

namespace coup {
namespace policy {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kRowThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLog2eLow = 1.925963033500576e-08f;  // what kLog2e rounds off
// Stands for -inf in products with a 0 share: 1e4 (the largest coefficient of
// the loss) times it is still finite.  Rows where a reference's logit is that
// far below its largest at an action with a share are taken again (far_row).
constexpr float kLowest = -1e33f;

template <class T>
__device__ __forceinline__ float widen(T v) {
  return (float)v;
}

// The rows of a call, as the kernels take them.
struct Rows {
  const void* logits;
  const void* ref;  // null: no reference policy
  int64_t stride, ref_stride;  // elements between rows
  const int8_t* actions;
  const uint32_t* mask;
  int64_t n;
  int A;
};

// The legal actions of a mask word among A: none at a chance node.
__device__ __forceinline__ uint32_t legal_bits(uint32_t mask, int A) {
  return (mask >> 31) ? 0u : mask & ((1u << A) - 1u);
}

__device__ __forceinline__ bool decided(uint32_t legal, int action) {
  return action >= 0 && action < 31 && ((legal >> action) & 1u);
}

// v where bit a of `legal` is set, else `other`: a field extract and a bit
// select (the compiler, seeing what m is, would make a test, a comparison and
// a conditional move of it).
__device__ __forceinline__ float keep(uint32_t legal, int a, float v, float other) {
  uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)legal, a, 1);
  asm("" : "+v"(m));
  return __uint_as_float((__float_as_uint(v) & m) | (__float_as_uint(other) & ~m));
}

// One row's legal word and action: no legal action, and action 0, where it
// does not count.
__device__ __forceinline__ uint32_t row_of(const Rows& r, int64_t i, bool mine, int& action) {
  const uint32_t legal = mine ? legal_bits(r.mask[i], r.A) : 0u;
  action = mine ? r.actions[i] : 0;
  if (decided(legal, action)) return legal;
  action = 0;
  return 0u;
}

// ------------------------------------------------- rows through the LDS
//
// A block's 256 rows are one run of memory when the table is contiguous, so
// its threads copy it in 16-byte pieces, all of them issued before the first
// is used, into LDS, and each thread then reads its own row from there (72
// bytes apart for the game's 18 float logits; read straight from memory those
// loads touch 64 lines an instruction: the 4 x 2^20-row loss took 461 us that
// way).  A gradient goes the same way back.  Strided tables are copied
// by elements.
//
// LDS: element j of row r is at byte (r A + j) sizeof(T), so a wave's lanes
// read words A sizeof(T) / 4 apart: for odd multiples of 4 or 8 bytes at most
// two lanes meet in a bank.  Rows that are multiples of 16 bytes (8, 16, 24
// float logits...) would meet 8 or 16 deep; they are read in 16-byte pieces,
// and piece k of the tile stands at place k ^ (k / 16 mod 16), which spreads
// one column of pieces over the 16 places.
template <class T, int AP>
struct Tile {
  static constexpr int kPieces = (AP * (int)sizeof(T) + 15) / 16;  // 16-byte pieces a thread, at most
  static constexpr int kBytes = kRowThreads * kPieces * 16 + 256;  // reads past a tile's last row stay inside
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
  // a piece in memory: at any element (gfx950's 16-byte accesses need no alignment)
  typedef uint32_t piece_at __attribute__((ext_vector_type(4), aligned(2)));

  // rows in whole pieces
  static __device__ __forceinline__ bool whole(int A) { return (A * (int)sizeof(T)) % 16 == 0; }
  static __device__ __forceinline__ int place(int k) { return k ^ ((k >> 4) & 15); }

  // The block's rows [row0, row0 + rows) in flight to registers.
  struct Flight {
    u32x4 piece[kPieces];
  };

  static __device__ __forceinline__ void fetch(Flight& f, const T* base, int64_t row0, int rows, int A) {
    const char* src = (const char*)(base + row0 * A);
    const int bytes = rows * A * (int)sizeof(T);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const uint32_t at = (c * kRowThreads + threadIdx.x) * 16;
      f.piece[c] = u32x4{0, 0, 0, 0};
      if ((int)at + 16 <= bytes) f.piece[c] = *(const piece_at*)(src + at);
    }
  }

  static __device__ __forceinline__ void land(const Flight& f, char* lds, const T* base, int64_t row0, int rows, int A) {
    const int bytes = rows * A * (int)sizeof(T);
    const bool w = whole(A);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const int k = c * kRowThreads + (int)threadIdx.x;
      if (k * 16 + 16 <= bytes) *(u32x4*)(lds + (w ? place(k) : k) * 16) = f.piece[c];
    }
    if (!w) {  // what is left of the last piece (whole rows leave none)
      const int k = bytes / 16 * 16 / (int)sizeof(T) + (int)threadIdx.x;
      if (k < rows * A) ((T*)lds)[k] = base[row0 * A + k];
    }
  }

  // LDS byte of element e of the tile
  static __device__ __forceinline__ int at_element(int e, int A) {
    const int b = e * (int)sizeof(T);
    return whole(A) ? place(b >> 4) * 16 + (b & 15) : b;
  }

  // The same through elements, for strided rows.
  static __device__ __forceinline__ void copy_in(char* lds, const T* base, int64_t stride, int64_t row0, int rows, int A) {
    const uint32_t inv = ((1u << 20) + A - 1) / A;  // e / A = e inv >> 20: e < 256 A, and e (A - 1) < 2^20
#pragma unroll 1
    for (int e = (int)threadIdx.x; e < rows * A; e += kRowThreads) {
      const int r = (int)((uint32_t)e * inv >> 20);
      *(T*)(lds + at_element(e, A)) = base[(row0 + r) * stride + (e - r * A)];
    }
  }

  // This thread's logit of one action.
  static __device__ __forceinline__ float read_one(const char* lds, int A, int action) {
    return widen(*(const T*)(lds + at_element((int)threadIdx.x * A + action, A)));
  }
  static __device__ __forceinline__ void write_one(char* lds, int A, int action, float g) {
    *(T*)(lds + at_element((int)threadIdx.x * A + action, A)) = (T)g;
  }

  // This thread's row, widened; -inf at actions outside `legal`.
  static __device__ __forceinline__ void read(const char* lds, int A, uint32_t legal, float (&x)[AP]) {
    const int r = (int)threadIdx.x;
    if (whole(A)) {
      const int k0 = r * A * (int)sizeof(T) / 16;
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const vec v = *(const vec*)(lds + place(k0 + c) * 16);
#pragma unroll
        for (int j = 0; j < (int)(16 / sizeof(T)); ++j) {
          const int a = c * (int)(16 / sizeof(T)) + j;
          if (a < AP) x[a] = widen((T)v[j]);
        }
      }
    } else if (sizeof(T) == 2 && !(A & 1)) {
      typedef T two __attribute__((ext_vector_type(2)));
      const two* row = (const two*)(lds + r * A * (int)sizeof(T));
#pragma unroll
      for (int a = 0; a < AP; a += 2) {
        const two v = row[a / 2];
        x[a] = widen((T)v[0]);
        x[a + 1] = widen((T)v[1]);
      }
    } else {
      const T* row = (const T*)lds + r * A;
#pragma unroll
      for (int a = 0; a < AP; ++a) x[a] = widen(row[a]);
    }
    // The masks are made here, not kept from another table's, and used here,
    // not carried beside the raw logits to where x is.
    asm volatile("" : "+v"(legal));
#pragma unroll
    for (int a = 0; a < AP; ++a) {
      x[a] = keep(legal, a, x[a], -INFINITY);
      asm volatile("" : "+v"(x[a]));
    }
  }

  // This thread's row of results, rounded, over its row.
  static __device__ __forceinline__ void write(char* lds, int A, const float (&g)[AP]) {
    const int r = (int)threadIdx.x;
    if (whole(A)) {
      const int k0 = r * A * (int)sizeof(T) / 16;
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        vec v;
#pragma unroll
        for (int j = 0; j < (int)(16 / sizeof(T)); ++j) {
          const int a = c * (int)(16 / sizeof(T)) + j;
          v[j] = (T)(a < AP ? g[a < AP ? a : 0] : 0.0f);
        }
        if (c * (int)(16 / sizeof(T)) < A) *(vec*)(lds + place(k0 + c) * 16) = v;
      }
    } else if (sizeof(T) == 2 && !(A & 1)) {
      typedef T two __attribute__((ext_vector_type(2)));
      two* row = (two*)(lds + r * A * (int)sizeof(T));
#pragma unroll
      for (int a = 0; a < AP; a += 2)
        if (a < A) row[a / 2] = two{(T)g[a], (T)g[a + 1]};
    } else {
      T* row = (T*)lds + r * A;
#pragma unroll
      for (int a = 0; a < AP; ++a)
        if (a < A) row[a] = (T)g[a];
    }
  }

  // The tile's rows out to a contiguous table.
  static __device__ __forceinline__ void copy_out(const char* lds, T* base, int64_t row0, int rows, int A) {
    const int n = rows * A, bytes = n * (int)sizeof(T);
    T* dst = base + row0 * A;
    const bool w = whole(A);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const int k = c * kRowThreads + (int)threadIdx.x;
      if (k * 16 + 16 <= bytes) *(piece_at*)((char*)dst + (uint32_t)k * 16) = *(const u32x4*)(lds + (w ? place(k) : k) * 16);
    }
    const int e = bytes / 16 * 16 / (int)sizeof(T) + (int)threadIdx.x;  // the last piece's rest (none of whole rows)
    if (e < n) dst[e] = ((const T*)lds)[e];
  }
};

// A block's rows of a table into LDS (its own: the caller keeps other
// threads' uses of it apart with barriers).
template <class T, int AP>
__device__ __forceinline__ void stage(char* lds, const void* base, int64_t stride, int64_t row0, int rows, int A) {
  using Tl = Tile<T, AP>;
  if (stride == A) {
    typename Tl::Flight f;
    Tl::fetch(f, (const T*)base, row0, rows, A);
    Tl::land(f, lds, (const T*)base, row0, rows, A);
  } else {
    Tl::copy_in(lds, (const T*)base, stride, row0, rows, A);
  }
}

// A block's rows, and (REF) its reference's before them, through one tile:
// both are in flight before the first is waited for, and `reference`, called
// on the reference's row d and its logit of `action`, works while the other
// still flies.  Then x and xa are the logits' own.  `action` must be one of
// the A (0 for rows that do not count).
template <class T, int AP, bool REF, class F>
__device__ __forceinline__ void stage_rows(char* lds, const Rows& q, int64_t row0, int rows, uint32_t legal, int action,
                                           float (&d)[AP], F reference, float (&x)[AP], float& xa) {
  using Tl = Tile<T, AP>;
  if (REF) {
    typename Tl::Flight f;
    const bool pieces = q.stride == q.A && q.ref_stride == q.A;
    if (pieces) {
      typename Tl::Flight g;
      Tl::fetch(g, (const T*)q.ref, row0, rows, q.A);
      Tl::fetch(f, (const T*)q.logits, row0, rows, q.A);
      Tl::land(g, lds, (const T*)q.ref, row0, rows, q.A);
    } else {
      Tl::copy_in(lds, (const T*)q.ref, q.ref_stride, row0, rows, q.A);
    }
    __syncthreads();
    Tl::read(lds, q.A, legal, d);
    reference(d, Tl::read_one(lds, q.A, action));
    __syncthreads();
    if (pieces) Tl::land(f, lds, (const T*)q.logits, row0, rows, q.A);
    else Tl::copy_in(lds, (const T*)q.logits, q.stride, row0, rows, q.A);
  } else {
    stage<T, AP>(lds, q.logits, q.stride, row0, rows, q.A);
  }
  __syncthreads();
  Tl::read(lds, q.A, legal, x);
  xa = Tl::read_one(lds, q.A, action);
}

// The larger; NaN where either is (one instruction, and for three values too).
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The hardware's base-2 logarithm, exponential and reciprocal, each good to
// a unit in the last place.
__device__ __forceinline__ float log_of(float v) { return __builtin_amdgcn_logf(v) * kLn2; }  // v >= 1, or of a ratio
__device__ __forceinline__ float exp_of(float v) {  // the product's rounding, and the constant's, are made good
  const float hi = v * kLog2e, lo = __builtin_fmaf(v, kLog2eLow, __builtin_fmaf(v, kLog2e, -hi));
  const float e = __builtin_amdgcn_exp2f(hi);
  return e > 0.0f && e < INFINITY ? __builtin_fmaf(e * lo, kLn2, e) : e;  // 0 and inf as they are, whatever lo is
}
// log(1 + v), v > -1 / 2: the rounding of w = 1 + v is made good by v / (w - 1),
// along which log(w) / (w - 1) hardly changes.
__device__ __forceinline__ float log1p_of(float v) {
  const float w = 1.0f + v, d = w - 1.0f;
  return d == 0.0f ? v : log_of(w) * (v * __builtin_amdgcn_rcpf(d));
}

// log(1 + v) for any v > -1, and the log of a ratio near 1.
__device__ __forceinline__ float log1p_any(float v) { return v > -0.5f ? log1p_of(v) : log_of(1.0f + v); }
__device__ __forceinline__ float log_ratio(float a, float b) { return log1p_any((a - b) / b); }

struct Softmax {
  float m;    // largest logit
  float sum;  // sum of e
  float others;  // sum of the e's fractions, that is without the ones (PRECISE alone)
  float lse;  // log of the sum (PRECISE alone): log p_a = (x_a - m) - lse
  __device__ __forceinline__ float e(float logit) const { return __builtin_amdgcn_exp2f((logit - m) * kLog2e); }
  __device__ __forceinline__ float t(float logit) const { return max_of(logit - m, kLowest); }
  // The sum without one of the e's: 1 - p_a is rest / sum, which keeps its
  // digits where p_a is nearly 1 (its e is 1 and the only one).  PRECISE alone.
  __device__ __forceinline__ float rest(float one) const { return one == 1.0f && sum - others < 1.5f ? others : sum - one; }
};

template <int AP>
__device__ __forceinline__ float row_max(const float (&x)[AP]) {
  float m = x[0];
#pragma unroll
  for (int a = 1; a < AP; ++a) m = max_of(m, x[a]);
  return m;
}

// The log of a row's sum of e, `others` the sum of the e's fractions, that is
// without the ones: log1p of it while only one e is (near) 1, so that a nearly
// certain action's log probability keeps its precision.
__device__ __forceinline__ float lse_of(float sum, float others) {
  return sum - others < 1.5f ? log1p_of(others) : log_of(sum);
}

// e = exp(x - m), and x becomes t = x - m held above -inf, so that e t is 0
// where e is; a NaN or +inf logit makes the sum NaN.  The sum is at least 1,
// the largest logit's own e.  PRECISE: also others and lse.
template <bool PRECISE, int AP>
__device__ __forceinline__ Softmax softmax(float (&x)[AP], float (&e)[AP]) {
  Softmax s;
  s.m = row_max<AP>(x);
  s.sum = 0.0f;
  s.others = 0.0f;
#pragma unroll
  for (int a = 0; a < AP; ++a) {
    e[a] = s.e(x[a]);
    x[a] = s.t(x[a]);
    s.sum += e[a];
    if (PRECISE) s.others += __builtin_amdgcn_fractf(e[a]);
  }
  s.lse = PRECISE ? lse_of(s.sum, s.others) : 0.0f;
  return s;
}

// This thread's row's sum of e in 64 bits, from its logits in the tile, for
// rows next to a border and for calls of few rows.
template <class T, int AP>
__device__ __forceinline__ double sum64(const char* tile, int A, uint32_t legal, float m) {
  double sum = 0.0;
#pragma unroll 1
  for (uint32_t b = legal; b; b &= b - 1)
    sum += exp((double)Tile<T, AP>::read_one(tile, A, __builtin_ctz(b)) - (double)m);
  return sum;
}

// The action a uniform number u falls on: the first legal a whose running
// sum passes u * total, in 64 bits; the last with a share where rounding
// leaves the total at or below it.
template <class T, int AP>
__device__ __forceinline__ int pick64(const char* tile, int A, uint32_t legal, float m, float u) {
  const double t = (double)u * sum64<T, AP>(tile, A, legal, m);
  double c = 0.0;
  int last = -1;
#pragma unroll 1
  for (uint32_t b = legal; b; b &= b - 1) {
    const int a = __builtin_ctz(b);
    const double e = exp((double)Tile<T, AP>::read_one(tile, A, a) - (double)m);
    c += e;
    if (e > 0.0) last = a;
    if (c > t) return a;
  }
  return last;
}

// ------------------------------------------------------- action sampling

// Row i's action is min {a : sum_{b <= a} e_b > u total} (inverse
// distribution function over the legal actions in ascending order).  The
// 32-bit running sums are off by less than 2^-17 of the total: the e's
// relative error is (1 + |x - m|) 2^-23, which weighs at most 3 * 2^-23 over
// a row, and 31 additions and the product add 16 * 2^-23 a side.  A running
// sum that near to u * total sends the row through pick64.
// 2^20 bf16 rows (51 MB, much of it from the cache) take 14.3 us, 3.6 TB/s;
// the 356 vector instructions a wave would take 9 alone.  One row: 2.5 us.
constexpr float kPickMargin = 7.62939453125e-6f;  // 2^-17

template <class T, int AP>
__global__ __launch_bounds__(kRowThreads) void k_sample(Rows r, const float* __restrict__ uniform,
                                                         int8_t* __restrict__ actions, float* __restrict__ log_probs) {
  __shared__ __align__(16) char lds[Tile<T, AP>::kBytes];
  const int64_t row0 = (int64_t)blockIdx.x * kRowThreads, i = row0 + threadIdx.x;
  const int rows = (int)(r.n - row0 < kRowThreads ? r.n - row0 : kRowThreads);
  const bool mine = (int)threadIdx.x < rows;
  const uint32_t legal = mine ? legal_bits(r.mask[i], r.A) : 0u;
  float u = mine ? uniform[i] : 0.0f;
  stage<T, AP>(lds, r.logits, r.stride, row0, rows, r.A);
  __syncthreads();
  int action = -1;
  float logp = 0.0f;
  if (legal) {
    float x[AP], e[AP];
    Tile<T, AP>::read(lds, r.A, legal, x);
    const Softmax s = softmax<true, AP>(x, e);
    if (s.sum == s.sum) {
      bool near = !(u < 1.0f);  // outside [0, 1): below as 0, above (and a NaN) the last action with a share
      u = u < 0.0f ? 0.0f : u;
      const float t = u * s.sum;
      float c = 0.0f, gap = INFINITY;
      action = 0;  // the actions whose running sums are no more than t
#pragma unroll
      for (int a = 0; a < AP; ++a) {
        c += e[a];
        gap = fminf(gap, fabsf(c - t));
        action += c <= t;
      }
      near |= gap <= kPickMargin * s.sum;
      if (near) action = pick64<T, AP>(lds, r.A, legal, s.m, u);
      logp = (Tile<T, AP>::read_one(lds, r.A, action) - s.m) - s.lse;
    } else {
      logp = s.sum;  // NaN or +inf at a legal action: no distribution, no action
    }
  }
  if (mine) {
    actions[i] = (int8_t)action;
    if (log_probs) log_probs[i] = logp;
  }
}

// ------------------------------------------------------------ advantages

// Player p's advantage at its decision in step t is, with V its value there,
//   A = R + gamma V' - V + gamma lam A',
// R the rewards it gets from t until its next decision, V' and A' that
// decision's.  Back in time with z_p = R + gamma V' + gamma lam A' so far:
// a step adds its reward to every z_p; the step's player takes A = z_p - V
// and leaves z_p = gamma lam z_p + gamma (1 - lam) V for its earlier ones; a
// LAST or FIRST step cuts what lies behind it (z = 0 before its reward).
//
// A step's map of z_p is affine with factors of at most 1, so a stretch of
// steps is one pair (f, g), z -> f z + g, per player, and stretches compose.
// A factor of 0 (a cut) takes nothing of z, be it infinite or NaN.
// A block holds L lanes; its NT / L threads of a lane take kStretch steps
// each, latest first, all loaded before the first is used; a scan over the
// stretches' pairs gives each its z, and the block goes on to the next round of
// NT / L * kStretch steps.
//
// Where the lanes are too few to fill the chip, a long window is split over
// blocks too (grid y).  A block finds z behind its part by reading on: it
// composes the rounds that follow until no player's pair lets anything pass
// (games end: mostly one or two rounds; else to the window's end) and stores
// nothing there.  No block waits for another, and nothing is kept between two
// launches.
// 20 steps x 2^20 lanes of 6 players (390 MB) take 91 us, 4.2 TB/s, with 96
// vector instructions a wave and step (50 us alone); 64 x 65,536 of 2 (67 MB)
// 14.3 us, 4.7 TB/s; 4096 x 33, whose games end after some 25 steps, 8.5 us: a
// round read, a round computed, each a latency.
struct AdvantageArgs {
  const int8_t* rewards;  // [T][B][P]
  const uint8_t* step_type;
  const int8_t* players;
  const void* values;
  const void* bootstrap;  // [B][P] or null
  float *adv, *target;
  int64_t T, B;
  int64_t part;  // steps a block: a number of rounds
  int dtype;
  float gamma, gl, gv;  // gamma, gamma lam, gamma (1 - lam)
};

constexpr int kStretch = 8;

// A value as it is stored (16 or 32 bits), and widened.
__device__ __forceinline__ uint32_t load_bits(const void* p, int64_t i, int dtype) {
  return dtype == COUP_DTYPE_F32 ? ((const uint32_t*)p)[i] : (uint32_t)((const uint16_t*)p)[i];
}
__device__ __forceinline__ float widen_bits(uint32_t v, int dtype) {
  if (dtype == COUP_DTYPE_F32) return __uint_as_float(v);
  if (dtype == COUP_DTYPE_BF16) return __uint_as_float(v << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)v);
}

// P reward bytes of one step and lane, at any alignment.
template <int P>
struct Rewards {
  struct __attribute__((packed, aligned(1))) U32 { uint32_t v; };
  struct __attribute__((packed, aligned(1))) U16 { uint16_t v; };
  uint32_t lo = 0, hi = 0;
  __device__ __forceinline__ void load(const int8_t* p) {
    if (P >= 4) lo = ((const U32*)p)->v;
    if (P == 6) hi = ((const U16*)(p + 4))->v;
    if (P == 5) hi = (uint8_t)p[4];
    if (P == 2 || P == 3) lo = ((const U16*)p)->v;
    if (P == 3) hi = (uint8_t)p[2];
  }
  __device__ __forceinline__ float of(int p) const {
    const uint32_t w = (P == 3) ? (p < 2 ? lo : hi) : (p < 4 ? lo : hi);
    const int at = (P == 3) ? (p & 1) * (p < 2) : (p & 3);
    return (float)(int8_t)(w >> (8 * at));
  }
};

// A thread's steps in memory: step k of lane l is at uniform element `base[k]`
// plus `off[k]`.  With one stretch a lane the step is the block's, so the
// offset is the lane; with more, it is the lane and the stretch's steps from
// the round's first: below 2^17 lanes x 32 steps, or 2^15 x 64, 2^14 x 128, 2^11
// x 512, x 24 bytes of any array (launch_advantages_of).
template <int C>
struct Steps {
  int64_t base[C == 1 ? kStretch : 1];
  uint32_t off[C == 1 ? 1 : kStretch];
  template <class V>
  __device__ __forceinline__ V* at(V* p, int k, int scale = 1) const {
    const int64_t u = base[C == 1 ? k : 0] * scale;
    const uint32_t v = off[C == 1 ? 0 : k] * (uint32_t)(scale * sizeof(V));
    return (V*)((char*)(p + u) + v);
  }
};

// f z + g, and g where f is 0, whatever z.
__device__ __forceinline__ float join(float f, float z, float g) { return __builtin_fmaf(f, f != 0.0f ? z : 0.0f, g); }

// One stretch from its z: the outputs, and z after it.
template <int P, int C>
__device__ __forceinline__ void advance(const AdvantageArgs& q, const Steps<C>& at, const int (&st)[kStretch],
                                        const int (&pl)[kStretch], const Rewards<P> (&r)[kStretch],
                                        const float (&v)[kStretch], float (&z)[P], int steps) {
#pragma unroll
  for (int k = 0; k < kStretch; ++k) {
    const bool cut = !(st[k] & 1);
    const float gvv = q.gv * v[k];
    float target = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float here = (cut ? 0.0f : z[p]) + r[k].of(p), after = q.gl * here + gvv;
      const bool acts = p == pl[k];
      target = acts ? here : target;
      z[p] = acts ? after : here;
    }
    if (k < steps) {
      *at.at(q.adv, k) = pl[k] >= 0 ? target - v[k] : 0.0f;
      *at.at(q.target, k) = target;
    }
  }
}

template <int P, int L, int NT>
__global__ __launch_bounds__(NT) void k_advantages(AdvantageArgs q) {
  constexpr int C = NT / L;                // stretches of a lane in flight
  constexpr int CW = L < 64 ? 64 / L : 1;  // of them in a wave
  constexpr int NW = C / CW;               // waves a lane's stretches span
  constexpr int LW = L < 64 ? L : 64;
  constexpr int kSteps = C * kStretch;     // a round's
  constexpr bool PARTS = L < 64;           // blocks that share a window
  static_assert(C == 1 || L <= 64, "a wave's threads are of one run of lanes");
  __shared__ float totals[C > 1 ? NW * LW * P * 2 : 1];
  const int64_t b0 = (int64_t)blockIdx.x * L;
  const int lanes = (int)(q.B - b0 < L ? q.B - b0 : L);
  const int l = (int)threadIdx.x % L, c = (int)threadIdx.x / L;
  const int cw = c % CW, wave = c / CW;        // C > 1: this stretch in its wave
  const int lane = l < lanes ? l : lanes - 1;  // lanes past the last load its steps and store nothing

  // This thread's steps of [first, end), at most kSteps: kStretch back from step first + top; ones before the first
  // load it and are skipped.
  struct Round {
    Steps<C> at;
    int st[kStretch], pl[kStretch], top;
    Rewards<P> r[kStretch];
    float v[kStretch];
  };
  const auto load = [&](Round& o, int64_t first, int64_t end) {
    int top = (int)(end - first) - 1 - c * kStretch;
    if (PARTS) asm volatile("" : "+v"(top));  // else every round's addresses are kept from the first: twice the registers
    o.top = top;
#pragma unroll
    for (int k = 0; k < kStretch; ++k) {
      const int rel = top - k > 0 ? top - k : 0;
      if (C == 1) o.at.base[k < (int)(sizeof(o.at.base) / 8) ? k : 0] = (first + rel) * q.B + b0;
      else o.at.off[k < (int)(sizeof(o.at.off) / 4) ? k : 0] = (uint32_t)rel * (uint32_t)q.B + lane;
    }
    if (C == 1) o.at.off[0] = lane;
    else o.at.base[0] = first * q.B + b0;
    uint32_t bits[kStretch];
#pragma unroll
    for (int k = 0; k < kStretch; ++k) {
      o.st[k] = *o.at.at(q.step_type, k);
      o.pl[k] = *o.at.at(q.players, k);
      o.r[k].load(o.at.at(q.rewards, k, P));
    }
    if (q.dtype == COUP_DTYPE_F32) {
#pragma unroll
      for (int k = 0; k < kStretch; ++k) bits[k] = *o.at.at((const uint32_t*)q.values, k);
    } else {
#pragma unroll
      for (int k = 0; k < kStretch; ++k) bits[k] = *o.at.at((const uint16_t*)q.values, k);
    }
#pragma unroll
    for (int k = 0; k < kStretch; ++k) {
      // FIRST 0 and LAST 2 cut, MID 1 and LAST 2 are steps; the rest is skipped, as 3
      o.st[k] = k > top || o.st[k] > COUP_STEP_SKIPPED ? COUP_STEP_SKIPPED : o.st[k];
      const bool step = o.st[k] == COUP_STEP_MID || o.st[k] == COUP_STEP_LAST;
      o.r[k].lo = step ? o.r[k].lo : 0u;
      o.r[k].hi = step ? o.r[k].hi : 0u;
      o.pl[k] = step && o.pl[k] < P ? o.pl[k] : -1;
      o.v[k] = o.pl[k] >= 0 ? widen_bits(bits[k], q.dtype) : 0.0f;
    }
  };
  // Its stretch's pairs (f, g), composed with those before it in its wave; the waves' wholes go to `totals`.
  const auto compose = [&](const Round& o, float (&f)[P], float (&g)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) f[p] = 1.0f, g[p] = 0.0f;
#pragma unroll
    for (int k = 0; k < kStretch; ++k) {
      const bool cut = !(o.st[k] & 1);
      const float gvv = q.gv * o.v[k];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const float here = (cut ? 0.0f : g[p]) + o.r[k].of(p), after = q.gl * here + gvv;
        const bool acts = p == o.pl[k];
        const float kept = cut ? 0.0f : f[p];
        f[p] = acts ? q.gl * kept : kept;
        g[p] = acts ? after : here;
      }
    }
    // the wave's stretches up to each, a lower index (a later time) first
#pragma unroll
    for (int d = 1; d < CW; d *= 2) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const float f0 = __shfl_up(f[p], d * L, 64), g0 = __shfl_up(g[p], d * L, 64);
        if (cw >= d) {
          g[p] = join(f[p], g0, g[p]);
          f[p] *= f0;
        }
      }
    }
    if (cw == CW - 1) {
      float* mine = totals + (wave * LW + (l & (LW - 1))) * P * 2;
#pragma unroll
      for (int p = 0; p < P; ++p) mine[2 * p] = f[p], mine[2 * p + 1] = g[p];
    }
  };
  const auto total = [&](int w, int p) { return totals + ((w * LW + (l & (LW - 1))) * P + p) * 2; };

  float z[P];
#pragma unroll
  for (int p = 0; p < P; ++p)
    z[p] = q.bootstrap ? q.gamma * widen_bits(load_bits(q.bootstrap, (b0 + lane) * P + p, q.dtype), q.dtype) : 0.0f;

  // this block's steps [last, begin)
  const int64_t begin = PARTS ? q.T - (int64_t)blockIdx.y * q.part : q.T;
  const int64_t last = PARTS && begin > q.part ? begin - q.part : 0;
  if (PARTS && begin < q.T) {
    // z behind them: the rounds after `begin` up to where nothing passes, or the window's end
    float F[P], G[P];
#pragma unroll
    for (int p = 0; p < P; ++p) F[p] = 1.0f, G[p] = 0.0f;
    for (int64_t first = begin; first < q.T; first += kSteps) {
      Round o;
      float f[P], g[P];
      load(o, first, first + kSteps);
      compose(o, f, g);
      __syncthreads();
      bool passes = false;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float a = 1.0f, b = 0.0f;
        for (int w = 0; w < NW; ++w) {
          const float* whole = total(w, p);
          b = join(whole[0], b, whole[1]);
          a *= whole[0];
        }
        G[p] = join(F[p], b, G[p]);
        F[p] *= a;
        passes |= F[p] != 0.0f;
      }
      if (!__syncthreads_or(passes)) break;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) z[p] = join(F[p], z[p], G[p]);
  }

  for (int64_t end = begin; end > last; end -= kSteps) {
    Round o;
    load(o, end > kSteps ? end - kSteps : 0, end);
    const int steps = l < lanes ? o.top + 1 : 0;
    if (C == 1) {
      advance<P, C>(q, o.at, o.st, o.pl, o.r, o.v, z, steps);
    } else {
      float f[P], g[P];
      compose(o, f, g);
      // what stands before this stretch in its wave
#pragma unroll
      for (int p = 0; p < P; ++p) {
        f[p] = CW > 1 ? __shfl_up(f[p], L, 64) : 1.0f;
        g[p] = CW > 1 ? __shfl_up(g[p], L, 64) : 0.0f;
        if (cw == 0) f[p] = 1.0f, g[p] = 0.0f;
      }
      __syncthreads();
      float here[P];
      for (int w = 0; w < NW; ++w) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const float* whole = total(w, p);
          if (w == wave) here[p] = join(f[p], z[p], g[p]);  // z runs through the waves: here it stands before this one
          z[p] = join(whole[0], z[p], whole[1]);
        }
      }
      __syncthreads();  // the next round writes the totals again
      advance<P, C>(q, o.at, o.st, o.pl, o.r, o.v, here, steps);
    }
  }
}

// ----------------------------------------------------- sums over a block

// v summed over the wave, in every lane: row shifts, then row broadcasts
// leave the sum in the last lane (no LDS traffic, six additions).
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_moved(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = add_moved<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = add_moved<0x112, 0xf>(v);
  v = add_moved<0x114, 0xf>(v);
  v = add_moved<0x118, 0xf>(v);
  v = add_moved<0x142, 0xa>(v);  // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  v = add_moved<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double add_moved(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xf, true);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The same in 64 bits, in the last lane alone.
__device__ __forceinline__ double wave_sum_last(double v) {
  v = add_moved<0x111, 0xf>(v);
  v = add_moved<0x112, 0xf>(v);
  v = add_moved<0x114, 0xf>(v);
  v = add_moved<0x118, 0xf>(v);
  v = add_moved<0x142, 0xa>(v);
  return add_moved<0x143, 0xc>(v);
}

// Four values summed over the wave at once, in 64 bits (a loss's terms nearly
// cancel): the sum of value k is lane k's (7 exchanges for 24: each of the first two halves what a lane still holds).
__device__ __forceinline__ double wave_sum_four(const float (&v)[4]) {
  const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
  const double a = (double)(odd ? v[1] : v[0]) + (double)__shfl_xor(odd ? v[0] : v[1], 1, 64);
  const double b = (double)(odd ? v[3] : v[2]) + (double)__shfl_xor(odd ? v[2] : v[3], 1, 64);
  double s = (upper ? b : a) + __shfl_xor(upper ? a : b, 2, 64);
#pragma unroll
  for (int d = 4; d < 64; d *= 2) s += __shfl_xor(s, d, 64);
  return s;
}

// Each of v[0..K) summed over the block, in a fixed order; thread 0 has the
// sums.  lds: K THREADS / 64 values.
template <int THREADS, int K, class V>
__device__ __forceinline__ void block_sum(V (&v)[K], V* lds) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v[k] += __shfl_xor(v[k], s, 64);
    if ((threadIdx.x & 63) == 0) lds[k * (THREADS / 64) + (threadIdx.x >> 6)] = v[k];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 0; k < K; ++k) {
      v[k] = 0;
      for (int w = 0; w < THREADS / 64; ++w) v[k] += lds[k * (THREADS / 64) + w];
    }
  }
}

// ----------------------------------------------------------- policy loss

// A decision's terms, with l = log pi, d = l - log pi_ref, rho =
// exp(l_action - old), the advantage Z and H = -sum p l, K = sum p d:
//   surrogate  -min(rho Z, clip(rho, 1 - low, 1 + high) Z)
//   loss       surrogate + kl K - ent H, averaged over the decisions.
// Its derivative in x_b, with w = -rho Z where the clip does not hold (else 0):
//   w ([b = action] - p_b) + p_b (kl (d_b - K) + ent (l_b + H)).
struct PolicyArgs {
  Rows r;
  const float* old;
  const float* adv;
  const uint8_t* active;  // null: every row
  double low, high;           // 1 - clip_low, 1 + clip_high
  float log_low, log_high;    // their logs
  float kl, ent;
  int few;  // ratios and log probabilities from 64-bit sums in every row (kFewRows)
  float* log_probs;  // null: not wanted
  void* grad;        // null: no gradient
  const float* grad_scale;  // its factor; null: 1
  double* partial;   // [blocks][4] sums of the terms over a block's rows
  int32_t* decided;  // [blocks] its decisions
  float* counts;     // [count blocks] the call's decisions, for the gradient
  uint32_t* ticket;  // of the folds that follow
  int count_blocks;
};

// Whether a row's t_ref (its held logits less their largest, softmax) is
// about kLowest at a legal action: the illegal ones alone add up to the rest.
template <int AP>
__device__ __forceinline__ bool is_far(const float (&t)[AP], uint32_t legal) {
  float sum = 0.0f;
#pragma unroll
  for (int a = 0; a < AP; ++a) sum += t[a];
  return sum < kLowest * ((float)(AP - __popc(legal)) + 0.5f);
}

// A row that is_far: one legal action's t_ref at least is below kLowest / 62.
// Where the policy takes such an action (with a share above 0 in 64 bits), K and
// the gradient (this thread's row of `tile`, if wanted) anew, in 64 bits and
// from memory.  K is infinite where the reference's logit is -inf, and then has
// no gradient: NaN at the legal actions.  Actions that both policies rule out
// (-inf, or a type's lowest value, in both) leave the row as it is.
template <class T, int AP>
__device__ __forceinline__ void far_row(const Rows& r, int64_t i, uint32_t legal, int action, double m, double rm, double w,
                                        double kl, double ent, double scale, bool grad, char* tile, float& K) {
  const T* x = (const T*)r.logits + i * r.stride;
  const T* ref = (const T*)r.ref + i * r.ref_stride;
  bool taken = false;
#pragma unroll 1
  for (uint32_t b = legal; b; b &= b - 1) {
    const int a = __builtin_ctz(b);
    taken |= (double)widen(x[a]) - m > -745.0 && (double)widen(ref[a]) - rm < (double)kLowest / 64;
  }
  if (!taken) return;
  double sum = 0.0, rsum = 0.0, et = 0.0, ed = 0.0;
#pragma unroll 1
  for (uint32_t b = legal; b; b &= b - 1) {
    const int a = __builtin_ctz(b);
    const double t = (double)widen(x[a]) - m, tr = (double)widen(ref[a]) - rm, e = exp(t);
    sum += e;
    rsum += exp(tr);
    et += e > 0.0 ? e * t : 0.0;
    ed += e > 0.0 ? e * (t - tr) : 0.0;
  }
  const double lse = log(sum), H = lse - et / sum, k = ed / sum - (lse - log(rsum));
  K = (float)k;
  if (!grad) return;
#pragma unroll 1
  for (uint32_t b = legal; b; b &= b - 1) {
    const int a = __builtin_ctz(b);
    const double t = (double)widen(x[a]) - m, tr = (double)widen(ref[a]) - rm, p = exp(t) / sum, l = t - lse;
    double g = w * ((a == action ? 1.0 : 0.0) - p);
    if (p > 0.0) g += p * (kl * (l - (tr - log(rsum)) - k) + ent * (l + H));
    if (!(k < INFINITY)) g = NAN;
    Tile<T, AP>::write_one(tile, r.A, a, (float)(g * scale));
  }
}

// Up to this many rows every row's ratio is taken in 64 bits, not only those
// by a border: a loss of few terms that nearly cancel keeps its digits (over
// many rows the 32-bit roundings average out).  A call of 65,536 float rows
// takes 14.6 us, one of 65,537 13.4.
constexpr int64_t kFewRows = 65536;
constexpr int kCountBlocks = 256, kCountThreads = 1024, kFinishThreads = 512;

// How many decisions there are: 6 bytes a row, four rows a thread at a time.
// The gradient needs it before its first store, and a second pass over the
// gradient would cost 2 A sizeof(T) a row.  4 x 2^20 rows (25 MB) 7 us.
__global__ __launch_bounds__(kCountThreads) void k_policy_count(PolicyArgs q) {
  __shared__ int wave[kCountThreads / 64];
  int n = 0;  // a thread's rows: below 2^31 for any call
  const int64_t first = (int64_t)blockIdx.x * kCountThreads + threadIdx.x, step = (int64_t)gridDim.x * kCountThreads;
  const bool fours = ((uintptr_t)q.r.mask & 15) == 0 && ((uintptr_t)q.r.actions & 3) == 0 &&
                     ((uintptr_t)q.active & 3) == 0;
  const int64_t quads = fours ? q.r.n / 4 : 0;
  for (int64_t i = first; i < quads; i += step) {
    const u32x4 m = ((const u32x4*)q.r.mask)[i];
    const uint32_t a = ((const uint32_t*)q.r.actions)[i];
    const uint32_t on = q.active ? ((const uint32_t*)q.active)[i] : ~0u;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      n += decided(legal_bits(m[k], q.r.A), (int8_t)(a >> (8 * k))) && ((on >> (8 * k)) & 0xFF);
  }
  for (int64_t i = 4 * quads + first; i < q.r.n; i += step)
    n += decided(legal_bits(q.r.mask[i], q.r.A), q.r.actions[i]) && (!q.active || q.active[i]);
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) n += __shfl_xor(n, s, 64);
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x != 0) return;
  int64_t total = 0;
  for (int w = 0; w < kCountThreads / 64; ++w) total += wave[w];
  q.counts[blockIdx.x] = (float)total;
}

// Loss and gradient in one pass, a tile a block: the tables are read once and
// the gradient written once.  4 x 2^20 float rows with a reference (961 MB)
// take 177 us, 5.4 TB/s; 1.3 M bf16 rows (165 MB) 42 us, 3.9 TB/s, bound by
// what four blocks a CU keep in flight (970 vector instructions a wave are 32
// us of it).  Four is what up to 128 registers allow; held to five the compiler
// spills, and 1.3 M rows took 65 us for 52 a call.
template <class T, int AP, bool REF>
__global__ __launch_bounds__(kRowThreads, AP <= 20 ? 4 : 2) void k_policy_loss(PolicyArgs q) {
  __shared__ double lds[4 * (kRowThreads / 64)];
  __shared__ int decisions[kRowThreads / 64];
  __shared__ __align__(16) char tile[Tile<T, AP>::kBytes];
  const int64_t row0 = (int64_t)blockIdx.x * kRowThreads, i = row0 + threadIdx.x;
  const int rows = (int)(q.r.n - row0 < kRowThreads ? q.r.n - row0 : kRowThreads);
  const bool mine = (int)threadIdx.x < rows;
  // the decisions of the call: every wave adds the counting blocks' numbers
  // (as 32-bit floats: they scale the gradient)
  float count = 0.0f, factor = 1.0f;
  if (q.grad) {
    if (q.grad_scale) factor = *q.grad_scale;
#pragma unroll
    for (int k = 0; k < kCountBlocks; k += 64) {
      const int at = k + ((int)threadIdx.x & 63);
      if (at < q.count_blocks) count += q.counts[at];
    }
  }
  int action;
  uint32_t legal = row_of(q.r, i, mine, action);
  float old = 0.0f, adv = 0.0f;
  if (mine) {
    if (q.active && !q.active[i]) legal = 0;
    old = q.old[i];
    adv = q.adv[i];
  }
  float x[AP], d[AP], xa, rta = 0.0f;  // d: the reference's t, rta the action's
  bool far = false;
  Softmax rs{0.0f, 1.0f, 0.0f, 0.0f};
  stage_rows<T, AP, REF>(
      tile, q.r, row0, rows, legal, action, d,
      [&](float(&row)[AP], float one) {
        float unused[AP];
        rs = softmax<false, AP>(row, unused);
        rta = rs.t(one);
        far = is_far<AP>(row, legal);
      },
      x, xa);
  const float n = wave_sum(count), scale = factor / (n > 0.0f ? n : 1.0f);
  float surrogate = 0.0f, kl = 0.0f, entropy = 0.0f, clipped = 0.0f, logp = 0.0f, ga = 0.0f, m = 0.0f, w = 0.0f;
  if (legal) {
    // x becomes t
    float e[AP];
    const Softmax s = softmax<true, AP>(x, e);
    float et = 0.0f, ed = 0.0f;  // sums of e t and e (t - t_ref)
#pragma unroll
    for (int a = 0; a < AP; ++a) {
      et += e[a] * x[a];
      if (REF) ed += e[a] * (x[a] - d[a]);
    }
    const float inv = __builtin_amdgcn_rcpf(s.sum);
    et *= inv, ed *= inv;
    entropy = s.lse - et;
    if (REF) kl = ed - log_ratio(s.sum, rs.sum);
    m = s.m;
    logp = (xa - s.m) - s.lse;
    const float dl = logp - old, border = adv > 0.0f ? q.log_high : q.log_low;
    bool over = adv > 0.0f ? dl > border : dl < border;
    float rho = exp_of(dl);
    // 32 bits hold dl to a few 2^-23 of its terms
    if (q.few || fabsf(dl - border) <= 4.76837158e-7f * (4.0f + fabsf(xa - s.m) + fabsf(old))) {
      const double whole = sum64<T, AP>(tile, q.r.A, legal, s.m);
      const double top = exp((double)xa - (double)s.m - (double)old);
      over = adv > 0.0f ? top > q.high * whole : top < q.low * whole;
      rho = (float)(top / whole);
      // (whole - 1 has an error of 2^-53: from 2^-32 down the fractions' sum is the better one)
      if (q.few) logp = (xa - s.m) - (s.rest(1.0f) < 2.3283064e-10f ? s.lse : lse_of((float)whole, (float)(whole - 1.0)));
    }
    over = over && adv != 0.0f;
    surrogate = adv == 0.0f ? 0.0f : -(over ? (float)(adv > 0.0f ? q.high : q.low) : rho) * adv;
    clipped = over ? 1.0f : 0.0f;
    if (q.grad) {
      // p_b w_b, w_b = ent (l_b + H) + kl (d_b - K) - w, in which the lse's
      // cancel: (ent + kl) (t_b - E t) - kl (tr_b - E tr) - w
      w = (over || adv == 0.0f) ? 0.0f : -rho * adv;
      // (the factor, which has no bound, meets p_b and not the coefficients
      // that kLowest is held for)
      const float share = inv * scale, ct = REF ? q.ent + q.kl : q.ent, cr = REF ? q.kl : 0.0f;
      const float held = cr * (et - ed) - ct * et, base = held - w;
#pragma unroll
      for (int a = 0; a < AP; ++a) x[a] = (e[a] * share) * (ct * x[a] + (REF ? base - cr * d[a] : base));
      // the action's own: w (1 - p_a) apart, of the other actions' e
      const float ea = s.e(xa);
      ga = (ea * share) * (ct * s.t(xa) + (REF ? held - cr * rta : held)) + (w * s.rest(ea)) * share;
      if (!(fabsf(base) < 1e30f && fabsf(scale) < INFINITY)) {  // else 0 times them is 0 at the actions outside the word
#pragma unroll
        for (int a = 0; a < AP; ++a) x[a] = keep(legal, a, x[a], 0.0f);
      }
    }
  } else {
#pragma unroll
    for (int a = 0; a < AP; ++a) x[a] = 0.0f;
  }
  if (mine && q.log_probs) q.log_probs[i] = logp;
  if (q.grad) {
    Tile<T, AP>::write(tile, q.r.A, x);
    if (legal) Tile<T, AP>::write_one(tile, q.r.A, action, ga);
  }
  if (REF && far) far_row<T, AP>(q.r, i, legal, action, m, rs.m, w, q.kl, q.ent, scale, q.grad && q.kl != 0.0f, tile, kl);
  if (q.grad) {
    __syncthreads();
    Tile<T, AP>::copy_out(tile, (T*)q.grad, row0, rows, q.r.A);
  }
  const float sums[4] = {surrogate, kl, entropy, clipped};
  const double v = wave_sum_four(sums);
  if ((threadIdx.x & 63) < 4) lds[(threadIdx.x >> 6) * 4 + (threadIdx.x & 63)] = v;
  const int here = (int)__popcll(__ballot(legal != 0));
  if ((threadIdx.x & 63) == 0) decisions[threadIdx.x >> 6] = here;
  __syncthreads();
  if (threadIdx.x < 4) {
    double total = 0.0;
    for (int w = 0; w < kRowThreads / 64; ++w) total += lds[4 * w + threadIdx.x];
    q.partial[4 * (int64_t)blockIdx.x + threadIdx.x] = total;
  }
  if (blockIdx.x == 0 && threadIdx.x == 5) *q.ticket = 0;
  if (threadIdx.x == 4) {
    int total = 0;
    for (int w = 0; w < kRowThreads / 64; ++w) total += decisions[w];
    q.decided[blockIdx.x] = total;
  }
}

// The blocks' sums in a fixed order, in 64 bits: the loss and its terms'
// means.  16,384 blocks (4 x 2^20 rows) leave 576 KiB, which one block takes
// 13 us to read; so from kFoldsFrom on up to kFoldBlocks of them fold a stretch
// each, and the one that is done last (by a ticket that the loss kernel reset)
// folds those, in 8 us.  1025 blocks: one block makes a call of 13.5 us, four
// 15.5; 5120: twenty fold in 5.8 us, five in 6.5.
constexpr int kFoldBlocks = 64, kFoldStretch = 256, kFoldsFrom = 2048;

__global__ __launch_bounds__(kRowThreads) void k_policy_finish(const double* __restrict__ partial,
                                                                const int32_t* __restrict__ decided, int64_t blocks,
                                                                double* fold, uint32_t* ticket, double kl, double ent,
                                                                float* loss, float* stats, int64_t* count) {
  __shared__ double lds[5 * (kRowThreads / 64)];
  __shared__ bool last;
  double s[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
  const int64_t from = blocks * blockIdx.x / gridDim.x, to = blocks * (blockIdx.x + 1) / gridDim.x;
  for (int64_t i = from + threadIdx.x; i < to; i += kRowThreads) {
#pragma unroll
    for (int k = 0; k < 4; ++k) s[k] += partial[4 * i + k];
    s[4] += (double)decided[i];
  }
  block_sum<kRowThreads, 5>(s, lds);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      for (int k = 0; k < 5; ++k) fold[5 * blockIdx.x + k] = s[k];
      __threadfence();  // the fold before the ticket, and the ticket before the others' folds
      last = atomicAdd(ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
    __syncthreads();
    if (!last) return;
#pragma unroll
    for (int k = 0; k < 5; ++k) s[k] = threadIdx.x < gridDim.x ? fold[5 * threadIdx.x + k] : 0.0;
    __syncthreads();
    block_sum<kRowThreads, 5>(s, lds);
  }
  if (threadIdx.x != 0) return;
  const double n = s[4] > 0.0 ? s[4] : 1.0;
  for (int k = 0; k < 4; ++k) s[k] /= n;
  *loss = (float)(s[0] + (kl != 0.0 ? kl * s[1] : 0.0) - ent * s[2]);
  for (int k = 0; k < 4; ++k)
    if (stats) stats[k] = (float)s[k];
  if (count) *count = (int64_t)s[4];
}

// ------------------------------------------------------- preference loss

// Sequences are packed: sequence s holds rows [offsets[s], offsets[s + 1]),
// 2 i the chosen and 2 i + 1 the rejected one of pair i.  With R_s = beta
// times the sum of l - l_ref over its decisions and x = R_2i - R_2i+1, a pair
// costs -(1 - eps) log sigma(x) - eps log sigma(-x); a row's derivative is
// +-beta / pairs (eps - sigma(-x)) ([b = action] - p_b).
struct PreferenceArgs {
  Rows r;
  const void* offsets;
  int wide;  // offsets are int64 (else int32)
  int64_t pairs;
  double beta, eps;
  float* loss;
  float* rewards;   // [2 pairs] or null
  void* grad;       // or null
  const float* grad_scale;  // its factor; null: 1
  double* partial;  // [blocks] a block's pairs' costs
  int group;        // the short form: pairs a block
  // the long form
  int slices;     // of a sequence, summed by a block each
  float* ratio;   // [n] a row's l - l_ref
  double* sums;   // [2 pairs][slices]
  float* coef;    // [2 pairs]
};

__device__ __forceinline__ int64_t raw_offset(const PreferenceArgs& q, int64_t s) {
  return q.wide ? ((const int64_t*)q.offsets)[s] : (int64_t)((const int32_t*)q.offsets)[s];
}

// Held to the rows: every row read is one of the call's.
__device__ __forceinline__ int64_t held(int64_t o, int64_t n) { return o < 0 ? 0 : o > n ? n : o; }
__device__ __forceinline__ int64_t offset_at(const PreferenceArgs& q, int64_t s) { return held(raw_offset(q, s), q.r.n); }

// The sequence of row i: the last that starts at or before it (the non-empty
// one where several start there); -1 before the first, 2 pairs behind the last.
// Offsets that do not ascend give some sequence too, and a later row never an
// earlier one: searches of two rows part where the earlier one goes left.
__device__ __forceinline__ int64_t sequence_of(const PreferenceArgs& q, int64_t i) {
  int64_t lo = 0, hi = 2 * q.pairs + 1;  // offsets[lo - 1] <= i < offsets[hi]
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (offset_at(q, mid) <= i) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

// Whether rows [from, to) are sequences first..last's by that search.  Runs of
// rows that are belong to different sequences where they do not meet, so those
// that pass are together no more than the call's rows, whatever the offsets;
// of ascending offsets every run passes.  Asked for long runs alone: it takes
// some 20 loads one after another.
__device__ __forceinline__ bool owned(const PreferenceArgs& q, int64_t from, int64_t to, int64_t first, int64_t last) {
  return sequence_of(q, from) >= first && sequence_of(q, to - 1) <= last;
}
constexpr int kGroupTrusted = 1024, kSliceTrusted = 16384;  // rows of a run that is not asked for

// A pair from its sequences' summed log ratios: its cost, and coef, the
// derivative in a chosen row's log ratio (a rejected row's is -coef).  NaN
// where `ok` is false: its offsets do not ascend within the rows.  With
// y = exp(-|x|), -log sigma(+-x) is log(1 + y) and for the wrong sign |x| more,
// and sigma(-|x|) is y / (1 + y): 32 bits hold both to a few units.  x is
// infinite where one sequence holds an action of probability 0.
__device__ __forceinline__ float pair_cost(const PreferenceArgs& q, int64_t pair, double chosen, double rejected, bool ok,
                                           float* coef) {
  chosen *= q.beta, rejected *= q.beta;
  if (!ok) chosen = rejected = NAN;
  if (q.rewards) q.rewards[2 * pair] = (float)chosen, q.rewards[2 * pair + 1] = (float)rejected;
  const double whole = chosen - rejected;
  const float x = (float)whole, size = fabsf(x), eps = (float)q.eps;
  // what x lost to rounding: exp(-|x|) has its absolute error as a relative one
  const float less = size < INFINITY ? (float)(fabs(whole) - (double)size) : 0.0f;
  float y = exp_of(-size);
  y -= y * less;
  const float part = __builtin_amdgcn_rcpf(1.0f + y);
  const float miss = x > 0.0f ? y * part : part;  // sigma(-x)
  const float factor = q.grad_scale ? *q.grad_scale : 1.0f;
  *coef = ok ? (eps - miss) * (float)(q.beta / (double)q.pairs) * factor : NAN;
  const float wrong = x > 0.0f ? eps : 1.0f - eps;
  return ok ? log1p_of(y) + (wrong != 0.0f ? wrong * size : 0.0f) : NAN;  // an infinite x costs nothing without a weight
}

__device__ __forceinline__ bool ascending(int64_t a, int64_t b, int64_t c, int64_t n) {
  return a >= 0 && b >= a && c >= b && c <= n;
}

// A tile's rows: this thread's log ratio, its e, their sum, and that without the action's.
template <class T, int AP, bool REF, bool FEW>
__device__ __forceinline__ float row_ratio(char* tile, const PreferenceArgs& q, int64_t row0, int rows, uint32_t legal,
                                           int action, float (&e)[AP], float& rest, float& sum) {
  float x[AP], d[AP], xa, out = 0.0f, one = 0.0f;
  double whole = 1.0;
  Softmax rs{0.0f, 1.0f, 0.0f, 0.0f};
  stage_rows<T, AP, REF>(
      tile, q.r, row0, rows, legal, action, d,
      [&](float(&row)[AP], float taken) {
        float unused[AP];
        rs = softmax<false, AP>(row, unused);
        one = taken;
        if (FEW) whole = sum64<T, AP>(tile, q.r.A, legal, rs.m);  // the tile holds the reference's rows here
      },
      x, xa);
  sum = 1.0f;
  rest = 0.0f;
  if (legal) {
    const Softmax s = softmax<true, AP>(x, e);
    // the two sums' logs as one, of a ratio near 1
    out = REF ? (xa - s.m) - (one - rs.m) : xa - s.m;
    if (FEW) {
      out -= log1p_any((float)(sum64<T, AP>(tile, q.r.A, legal, s.m) / whole - 1.0));
    } else {
      out -= REF ? log_ratio(s.sum, rs.sum) : log_of(s.sum);
    }
    rest = s.rest(s.e(xa));
    sum = s.sum;
  }
  return out;
}

// The gradient of a tile's rows: coef ([b = action] - e_b / sum), the action's own as coef rest / sum.
template <class T, int AP>
__device__ __forceinline__ void row_grad(char* tile, const PreferenceArgs& q, int64_t row0, int rows, uint32_t legal,
                                         int action, float (&e)[AP], float rest, float sum, float coef) {
  const float p = -coef / sum;
#pragma unroll
  for (int a = 0; a < AP; ++a) e[a] = keep(legal, a, p * e[a], 0.0f);
  Tile<T, AP>::write(tile, q.r.A, e);
  if (legal) Tile<T, AP>::write_one(tile, q.r.A, action, -p * rest);
  __syncthreads();
  Tile<T, AP>::copy_out(tile, (T*)q.grad, row0, rows, q.r.A);
}

// Short sequences (a game's decisions): a block takes `group` consecutive
// pairs, whose rows are one run, mostly of one tile.  The tile is read once:
// its rows' log ratios go to LDS, a wave sums each sequence's, the pairs'
// costs follow, and the gradient is written from the e still in registers.
// A group of more rows goes through its tiles twice.  Blocks past the groups
// write the zero gradients of the rows outside every sequence.
// 8192 pairs over 327,680 bf16 rows (37 MB) take 24.7 us, bound by a block's
// latency: its steps wait for one another.  Groups of 120, 160 and 200 rows
// come to the same.
constexpr int kMaxGroup = 32, kZeroBlocks = 64;

template <class T, int AP, bool REF, bool FEW>
__global__ __launch_bounds__(kRowThreads, AP > 20 ? 2 : FEW ? 4 : sizeof(T) == 2 ? 6 : 5) void k_preference_short(PreferenceArgs q) {
  __shared__ __align__(16) char tile[Tile<T, AP>::kBytes];
  __shared__ float ratio[kRowThreads];
  __shared__ int64_t edge[2 * kMaxGroup + 1];
  __shared__ double sum[2 * kMaxGroup];
  __shared__ float coef[2 * kMaxGroup];
  const int64_t groups = (q.pairs + q.group - 1) / q.group;
  if ((int64_t)blockIdx.x >= groups) {
    if (!q.grad) return;
    // rows before the first sequence and behind the last, by elements
    const int64_t head = offset_at(q, 0) * q.r.A, tail = offset_at(q, 2 * q.pairs) * q.r.A, n = q.r.n * q.r.A;
    const int64_t first = ((int64_t)blockIdx.x - groups) * kRowThreads + threadIdx.x;
    for (int64_t k = first; k < head; k += (int64_t)kZeroBlocks * kRowThreads) ((T*)q.grad)[k] = (T)0.0f;
    for (int64_t k = tail + first; k < n; k += (int64_t)kZeroBlocks * kRowThreads) ((T*)q.grad)[k] = (T)0.0f;
    return;
  }
  const int64_t pair0 = (int64_t)blockIdx.x * q.group;
  const int pairs = (int)(q.pairs - pair0 < q.group ? q.pairs - pair0 : q.group);
  const int wave = (int)threadIdx.x >> 6, seqs = 2 * pairs;
  if ((int)threadIdx.x <= seqs) edge[threadIdx.x] = raw_offset(q, 2 * pair0 + threadIdx.x);
  if ((int)threadIdx.x < seqs) sum[threadIdx.x] = 0.0;
  __syncthreads();
  bool ok = true;
  if ((int)threadIdx.x < pairs) {
    const int64_t* o = edge + 2 * threadIdx.x;
    ok = ascending(o[0], o[1], o[2], q.r.n);
  }
  // a group of bad offsets is not walked, nor a long one that is not the rows' (offsets elsewhere do not ascend): the
  // groups walk 13 times the call's rows and 32 a pair at most
  bool good = __syncthreads_and(ok);
  if (good && edge[seqs] - edge[0] > kGroupTrusted)
    good = owned(q, edge[0], edge[seqs], 2 * pair0, 2 * pair0 + seqs - 1);
  const int64_t begin = good ? edge[0] : 0, end = good ? edge[seqs] : 0;

  // a tile's log ratios to its sequences' sums, in 64 bits (one pair's cost of e^-x has x's absolute error, and two
  // log ratios of a type's lowest logits pass 32 bits' range; 32-bit sums: 8192 bf16 pairs 24.6 us for 24.7)
  const auto add_tile = [&](int64_t row0, int rows) {
    __syncthreads();
    for (int s = wave; s < seqs; s += kRowThreads / 64) {
      const int64_t lo = edge[s] - row0, hi = edge[s + 1] - row0;
      const int to = !good ? 0 : hi < rows ? (int)hi : rows;
      double v = 0.0;
      for (int k = (lo > 0 ? (lo < rows ? (int)lo : rows) : 0) + ((int)threadIdx.x & 63); k < to; k += 64) v += (double)ratio[k];
      v = wave_sum_last(v);
      if ((threadIdx.x & 63) == 63) sum[s] += v;
    }
    __syncthreads();
  };
  // the pairs, lanes of one wave
  const auto close_pairs = [&]() {
    double cost = 0.0;
    if ((int)threadIdx.x < pairs) {
      const int s = 2 * threadIdx.x;
      cost = (double)pair_cost(q, pair0 + threadIdx.x, sum[s], sum[s + 1], good, &coef[s]);
      coef[s + 1] = -coef[s];
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int d = kMaxGroup / 2; d >= 1; d >>= 1) cost += __shfl_xor(cost, d, 64);
    if (threadIdx.x == 0) {
      q.partial[blockIdx.x] = cost;
      if (groups == 1) *q.loss = (float)(cost / (double)q.pairs);
    }
  };
  // the coef of row i: its sequence is the last that starts at or before it
  const auto coef_of = [&](int64_t i) {
    int lo = 0, hi = seqs;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (edge[mid + 1] <= i) lo = mid + 1;
      else hi = mid;
    }
    return lo < seqs ? coef[lo] : 0.0f;
  };

  float e[AP], rest, total;
  int action;
  if (end - begin <= kRowThreads) {
    const int64_t i = begin + threadIdx.x;
    const int rows = end > begin ? (int)(end - begin) : 0;
    const uint32_t legal = row_of(q.r, i, (int)threadIdx.x < rows, action);
    ratio[threadIdx.x] = row_ratio<T, AP, REF, FEW>(tile, q, begin, rows, legal, action, e, rest, total);
    add_tile(begin, rows);
    close_pairs();
    if (q.grad) row_grad<T, AP>(tile, q, begin, rows, legal, action, e, rest, total, coef_of(i));
    return;
  }
  for (int64_t row0 = begin; row0 < end; row0 += kRowThreads) {
    const int rows = (int)(end - row0 < kRowThreads ? end - row0 : kRowThreads);
    const uint32_t legal = row_of(q.r, row0 + threadIdx.x, (int)threadIdx.x < rows, action);
    ratio[threadIdx.x] = row_ratio<T, AP, REF, FEW>(tile, q, row0, rows, legal, action, e, rest, total);
    add_tile(row0, rows);
  }
  close_pairs();
  if (!q.grad) return;
  for (int64_t row0 = begin; row0 < end; row0 += kRowThreads) {
    const int64_t i = row0 + threadIdx.x;
    const int rows = (int)(end - row0 < kRowThreads ? end - row0 : kRowThreads);
    const uint32_t legal = row_of(q.r, i, (int)threadIdx.x < rows, action);
    stage<T, AP>(tile, q.r.logits, q.r.stride, row0, rows, q.r.A);
    __syncthreads();
    float x[AP];
    Tile<T, AP>::read(tile, q.r.A, legal, x);
    const float xa = Tile<T, AP>::read_one(tile, q.r.A, action);
    const Softmax sm = softmax<true, AP>(x, e);
    row_grad<T, AP>(tile, q, row0, rows, legal, action, e, sm.rest(sm.e(xa)), sm.sum, coef_of(i));
    __syncthreads();
  }
}

// Long sequences: every row's log ratio to memory, the sequences' sums from
// slices of them, the pairs, then the gradient with the logits read again
// (A sizeof(T) of a row's 3 A sizeof(T) + 5 bytes).  8 pairs over 1.5 M float
// rows: 35.0 us for the rows (229 MB, 6.5 TB/s, partly cached), 6.7 and 4.6 for
// the sums and pairs, 34.0 for the gradient (223 MB).
template <class T, int AP, bool REF, bool FEW>
__global__ __launch_bounds__(kRowThreads) void k_preference_rows(PreferenceArgs q) {
  __shared__ __align__(16) char tile[Tile<T, AP>::kBytes];
  const int64_t row0 = (int64_t)blockIdx.x * kRowThreads, i = row0 + threadIdx.x;
  const int rows = (int)(q.r.n - row0 < kRowThreads ? q.r.n - row0 : kRowThreads);
  const bool mine = (int)threadIdx.x < rows;
  int action;
  const uint32_t legal = row_of(q.r, i, mine, action);
  float e[AP], rest, total;
  const float out = row_ratio<T, AP, REF, FEW>(tile, q, row0, rows, legal, action, e, rest, total);
  if (mine) q.ratio[i] = out;
}

__global__ __launch_bounds__(kRowThreads) void k_preference_sums(PreferenceArgs q) {
  __shared__ double lds[kRowThreads / 64];
  const int64_t seq = (int64_t)blockIdx.x / q.slices;
  const int slice = (int)((int64_t)blockIdx.x % q.slices);
  const int64_t lo = offset_at(q, seq), hi = offset_at(q, seq + 1), len = hi > lo ? hi - lo : 0;
  const int64_t from = lo + len / q.slices * slice + (len % q.slices) * slice / q.slices;
  int64_t to = lo + len / q.slices * (slice + 1) + (len % q.slices) * (slice + 1) / q.slices;
  double s[1] = {0.0};
  // offsets that do not ascend: the slices walk some 200 times the call's rows at most
  if (to - from > kSliceTrusted && !owned(q, from, to, seq, seq)) to = from, s[0] = NAN;
#pragma unroll 4
  for (int64_t i = from + threadIdx.x; i < to; i += kRowThreads) s[0] += (double)q.ratio[i];
  block_sum<kRowThreads, 1>(s, lds);
  if (threadIdx.x == 0) q.sums[blockIdx.x] = s[0];
}

constexpr int kPairThreads = 1024, kPairsABlock = 64;

// A wave a pair: its slices' sums, its cost and coefs.
__global__ __launch_bounds__(kPairThreads) void k_preference_pairs(PreferenceArgs q) {
  __shared__ double lds[kPairThreads / 64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  double cost[1] = {0.0};
  for (int k = wave; k < kPairsABlock; k += kPairThreads / 64) {
    const int64_t pair = (int64_t)blockIdx.x * kPairsABlock + k;
    if (pair >= q.pairs) break;
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      for (int j = lane; j < q.slices; j += 64) s[h] += q.sums[(2 * pair + h) * q.slices + j];
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) s[h] += __shfl_xor(s[h], d, 64);
    }
    if (lane == 0) {
      const bool ok = ascending(raw_offset(q, 2 * pair), raw_offset(q, 2 * pair + 1), raw_offset(q, 2 * pair + 2), q.r.n);
      float d;
      cost[0] += (double)pair_cost(q, pair, s[0], s[1], ok, &d);
      q.coef[2 * pair] = d, q.coef[2 * pair + 1] = -d;
    }
  }
  block_sum<kPairThreads, 1>(cost, lds);
  if (threadIdx.x == 0) {
    q.partial[blockIdx.x] = cost[0];
    if (gridDim.x == 1) *q.loss = (float)(cost[0] / (double)q.pairs);
  }
}

template <class T, int AP>
__global__ __launch_bounds__(kRowThreads) void k_preference_grad(PreferenceArgs q) {
  __shared__ __align__(16) char tile[Tile<T, AP>::kBytes];
  const int64_t row0 = (int64_t)blockIdx.x * kRowThreads, i = row0 + threadIdx.x;
  const int rows = (int)(q.r.n - row0 < kRowThreads ? q.r.n - row0 : kRowThreads);
  int action;
  uint32_t legal = row_of(q.r, i, (int)threadIdx.x < rows, action);
  float coef = 0.0f;
  if (legal) {
    const int64_t seq = sequence_of(q, i);
    if (seq >= 0 && seq < 2 * q.pairs) coef = q.coef[seq];
    else legal = 0;
  }
  stage<T, AP>(tile, q.r.logits, q.r.stride, row0, rows, q.r.A);
  __syncthreads();
  float x[AP], e[AP];
  Tile<T, AP>::read(tile, q.r.A, legal, x);
  const float xa = Tile<T, AP>::read_one(tile, q.r.A, action);
  const Softmax sm = softmax<true, AP>(x, e);
  row_grad<T, AP>(tile, q, row0, rows, legal, action, e, sm.rest(sm.e(xa)), sm.sum, coef);
}

// The blocks' costs in a fixed order.
__global__ __launch_bounds__(kFinishThreads) void k_preference_finish(const double* __restrict__ partial, int64_t blocks,
                                                                       int64_t pairs, float* loss) {
  __shared__ double lds[kFinishThreads / 64];
  double s[1] = {0.0};
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < blocks; i += kFinishThreads) s[0] += partial[i];
  block_sum<kFinishThreads, 1>(s, lds);
  if (threadIdx.x == 0) *loss = (float)(s[0] / (double)(pairs > 0 ? pairs : 1));
}

// ---------------------------------------------------------- grad scaling

// A gradient for a loss's own derivative of 1, times the derivative that
// came in: nothing is read or written where that is 1, as in loss.backward()
// (1.9 us, a launch).  A second rounding, at most another half step; nothing
// for a power of two, unless the first one was to a half's smallest steps,
// which is what grad_scale is for.  What is 0 stays it, whatever came in.
template <class T>
__global__ __launch_bounds__(kRowThreads) void k_scale_grad(T* grad, int64_t n, const float* __restrict__ scale) {
  const float g = *scale;
  if (g == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kRowThreads)
    if (const float v = (float)grad[i]; v != 0.0f) grad[i] = (T)(g * v);
}

// ---------------------------------------------------------------- launch

inline unsigned row_blocks(int64_t n) { return (unsigned)((n + kRowThreads - 1) / kRowThreads); }

template <class T>
struct type_of {
  using type = T;
};

// f(type_of<T>, integral AP) for a dtype code and a number of actions: rows
// are padded to 8, 16, 20 or 32 actions (20: the game's 18).
template <class T, class F>
void with_actions(int A, F f) {
  if (A <= 8) f(type_of<T>(), std::integral_constant<int, 8>());
  else if (A <= 16) f(type_of<T>(), std::integral_constant<int, 16>());
  else if (A <= 20) f(type_of<T>(), std::integral_constant<int, 20>());
  else f(type_of<T>(), std::integral_constant<int, 32>());
}

template <class F>
void with_dtype(int dtype, F f) {
  if (dtype == COUP_DTYPE_F32) f(type_of<float>());
  else if (dtype == COUP_DTYPE_F16) f(type_of<_Float16>());
  else f(type_of<__bf16>());
}

template <class F>
void with_rows(int dtype, int A, F f) {
  with_dtype(dtype, [&](auto t) { with_actions<typename decltype(t)::type>(A, f); });
}

// f(bool constant, bool constant)
template <class F>
void with_flags(bool a, bool b, F f) {
  if (a && b) f(std::true_type(), std::true_type());
  else if (a) f(std::true_type(), std::false_type());
  else if (b) f(std::false_type(), std::true_type());
  else f(std::false_type(), std::false_type());
}

inline void launch_sample(const Rows& r, int dtype, const float* uniform, int8_t* actions, float* log_probs,
                          hipStream_t s) {
  with_rows(dtype, r.A, [&](auto t, auto ap) {
    using T = typename decltype(t)::type;
    k_sample<T, decltype(ap)::value><<<row_blocks(r.n), kRowThreads, 0, s>>>(r, uniform, actions, log_probs);
  });
}

// How a window is split: L lanes a block and C of each one's stretches at a
// time (few lanes a block read short runs of memory), by the lanes there are
// to fill the chip with and with no more stretches than the window has; then
// into parts, up to a block a CU (twice that: no faster), that look for their
// z themselves.  Either side of the borders, 2 players, games of some 25 steps,
// us, L x C: 256 steps x 65,536 lanes 64 x 4 52, 256 x 1 77; 256 x 131,072 256 x
// 1 117, 64 x 4 122; 512 x 32,768 64 x 4 54, 64 x 8 67; 1024 x 16,384 64 x 8
// 63, 64 x 4 86, 32 x 16 80; 512 x 8192 32 x 16 24.4, 64 x 8 29; 200 x 1500
// 8 x 32 6.6, 32 x 16 9.2; 500 x 1500 8 x 64 12.3, 32 x 16 13.8, 500 x 2100
// 17.0, 18.2; 4000 x 256 32 x 16 13.5, 8 x 32 17.7; 4000 x 130 15.9, 14.5.
// Without parts 1024 x 2048 took 35 for 18, 4096 x 33 16.7 for 8.5.  A window
// without one cut, whose parts all read on to its end, loses by them: 4096 x 33
// 39, 1024 x 2048 29.
constexpr int64_t kPartBlocks = 256;

template <int P, int L, int NT>
void launch_advantages_as(AdvantageArgs q, hipStream_t s) {
  constexpr int64_t kSteps = NT / L * kStretch;
  const int64_t groups = (q.B + L - 1) / L, rounds = (q.T + kSteps - 1) / kSteps;
  int64_t parts = L < 64 && groups < kPartBlocks ? kPartBlocks / groups : 1;
  if (parts > rounds) parts = rounds;
  q.part = (rounds + parts - 1) / parts * kSteps;
  const unsigned y = (unsigned)((q.T + q.part - 1) / q.part);
  k_advantages<P, L, NT><<<dim3((unsigned)groups, y), NT, 0, s>>>(q);
}

template <int P>
void launch_advantages_of(const AdvantageArgs& q, hipStream_t s) {
  const auto enough = [&](int c, int64_t lanes) { return q.B >= lanes || (int64_t)c * kStretch >= q.T; };
  if (enough(1, 1 << 17)) launch_advantages_as<P, 256, 256>(q, s);
  else if (enough(4, 1 << 15)) launch_advantages_as<P, 64, 256>(q, s);
  else if (enough(8, 1 << 14)) launch_advantages_as<P, 64, 512>(q, s);
  else if (enough(16, 1 << 11)) launch_advantages_as<P, 32, 512>(q, s);
  else if (q.T > 32 * kStretch && q.T <= 64 * kStretch) launch_advantages_as<P, 8, 512>(q, s);
  else if (q.T > 64 * kStretch && q.B >= 1 << 8) launch_advantages_as<P, 32, 512>(q, s);
  else launch_advantages_as<P, 8, 256>(q, s);
}

inline void launch_advantages(const AdvantageArgs& q, int players, hipStream_t s) {
  switch (players) {
    case 2: return launch_advantages_of<2>(q, s);
    case 3: return launch_advantages_of<3>(q, s);
    case 4: return launch_advantages_of<4>(q, s);
    case 5: return launch_advantages_of<5>(q, s);
    default: return launch_advantages_of<6>(q, s);
  }
}

inline size_t policy_workspace(int64_t n) {
  return sizeof(double) * (4 * (size_t)row_blocks(n) + 5 * kFoldBlocks) + sizeof(float) * (kCountBlocks + 1) +
         sizeof(int32_t) * row_blocks(n);
}

inline void launch_policy(PolicyArgs q, int dtype, double kl, double ent, float* loss, float* stats, int64_t* count,
                          void* workspace, hipStream_t s) {
  const unsigned blocks = row_blocks(q.r.n);
  const int64_t counters = (q.r.n + 4 * kCountThreads - 1) / (4 * kCountThreads);
  q.partial = (double*)workspace;
  double* fold = q.partial + 4 * (int64_t)blocks;
  q.counts = (float*)(fold + 5 * kFoldBlocks);
  q.ticket = (uint32_t*)(q.counts + kCountBlocks);
  q.decided = (int32_t*)(q.ticket + 1);
  q.few = q.r.n <= kFewRows;
  q.count_blocks = (int)(counters < kCountBlocks ? counters : kCountBlocks);
  if (blocks) {
    if (q.grad) k_policy_count<<<q.count_blocks, kCountThreads, 0, s>>>(q);
    with_rows(dtype, q.r.A, [&](auto t, auto ap) {
      using T = typename decltype(t)::type;
      constexpr int AP = decltype(ap)::value;
      if (q.r.ref) k_policy_loss<T, AP, true><<<blocks, kRowThreads, 0, s>>>(q);
      else k_policy_loss<T, AP, false><<<blocks, kRowThreads, 0, s>>>(q);
    });
  }
  const unsigned stretches = blocks < kFoldsFrom ? 1 : blocks / kFoldStretch;
  const unsigned folds = stretches < kFoldBlocks ? stretches : kFoldBlocks;
  k_policy_finish<<<folds, kRowThreads, 0, s>>>(q.partial, q.decided, blocks, fold, q.ticket, kl, ent, loss, stats, count);
}

// How a preference call is split.  Short where a pair has at most kShortRows
// rows on average: `group` pairs a block, some 5 / 8 of a tile so that few
// groups spill into a second; else a sequence's sum takes a block per 4096
// rows of the average one.
// Few rows' sums are taken in 64 bits, as the policy loss's (kFewRows): the
// short form's up to a quarter of them (16,384 rows 18.6 us, 16,385 13.8; at
// 65,536 it would be 21 for 15), the long form's up to all (20.2, 17.5).
// A short block has 32 pairs or 81 rows and more on average, a long sequence
// more than 80, so the calls the entries take (COUP_MAX_DECISIONS,
// COUP_MAX_PAIRS) launch fewer than 2^32 threads.  One sequence far longer than
// its call's average keeps one block busy, 256 of its rows at a time (2^20
// rows, 8192 pairs: 53 us; with one sequence of 65,536 rows 1290).
// On either side of kShortRows, 2^19 bf16 rows, us: 40 rows a pair short 35,
// long 66; 150 43, 44; 165 41, 43; 300 44, 40; 1000 103, 37.
constexpr int kShortRows = 160;

struct PreferencePlan {
  bool is_short, few;
  int group, slices;
  int64_t blocks;  // that leave a partial sum
};

inline PreferencePlan preference_plan(int64_t n, int64_t pairs) {
  PreferencePlan p{};
  const int64_t each = pairs ? n / pairs : 0;
  p.is_short = each <= kShortRows;
  p.few = n <= (p.is_short ? kFewRows / 4 : kFewRows);
  if (p.is_short) {
    const int64_t g = kShortRows / (each > 0 ? each : 1);
    p.group = (int)(g < kMaxGroup ? g : kMaxGroup);
    p.blocks = (pairs + p.group - 1) / p.group;
  } else {
    const int64_t sl = each / 2 / 4096;
    p.slices = (int)(sl < 1 ? 1 : sl > 256 ? 256 : sl);
    p.blocks = (pairs + kPairsABlock - 1) / kPairsABlock;
  }
  return p;
}

inline size_t preference_workspace(int64_t n, int64_t pairs) {
  const PreferencePlan p = preference_plan(n, pairs);
  const size_t partial = sizeof(double) * (p.blocks + 1);
  if (p.is_short) return partial;
  return partial + sizeof(double) * 2 * pairs * p.slices + sizeof(float) * (2 * pairs + n);
}

inline void launch_preference(PreferenceArgs q, int dtype, void* workspace, hipStream_t s) {
  const PreferencePlan p = preference_plan(q.r.n, q.pairs);
  q.partial = (double*)workspace;
  q.group = p.group;
  q.slices = p.slices;
  const unsigned tiles = row_blocks(q.r.n);
  with_rows(dtype, q.r.A, [&](auto t, auto ap) {
    using T = typename decltype(t)::type;
    constexpr int AP = decltype(ap)::value;
    if (p.is_short) {
      const int64_t grid = p.blocks + (q.grad && q.r.n ? kZeroBlocks : 0);
      if (grid) {
        with_flags(q.r.ref != nullptr, p.few, [&](auto ref, auto few) {
          k_preference_short<T, AP, decltype(ref)::value, decltype(few)::value>
              <<<(unsigned)grid, kRowThreads, 0, s>>>(q);
        });
      }
    } else {
      q.sums = q.partial + p.blocks + 1;
      q.coef = (float*)(q.sums + 2 * q.pairs * p.slices);
      q.ratio = q.coef + 2 * q.pairs;
      with_flags(q.r.ref != nullptr, p.few, [&](auto ref, auto few) {
        k_preference_rows<T, AP, decltype(ref)::value, decltype(few)::value><<<tiles, kRowThreads, 0, s>>>(q);
      });
      k_preference_sums<<<(unsigned)(2 * q.pairs * p.slices), kRowThreads, 0, s>>>(q);
      k_preference_pairs<<<(unsigned)p.blocks, kPairThreads, 0, s>>>(q);
      if (q.grad) k_preference_grad<T, AP><<<tiles, kRowThreads, 0, s>>>(q);
    }
    if (p.blocks != 1) k_preference_finish<<<1, kFinishThreads, 0, s>>>(q.partial, p.blocks, q.pairs, q.loss);
  });
}

inline void launch_scale(void* grad, int dtype, int64_t n, const float* scale, hipStream_t s) {
  const int64_t blocks = (n + kRowThreads - 1) / kRowThreads;
  with_dtype(dtype, [&](auto t) {
    using T = typename decltype(t)::type;
    k_scale_grad<T><<<(unsigned)(blocks < 2048 ? blocks : 2048), kRowThreads, 0, s>>>((T*)grad, n, scale);
  });
}

}  // namespace policy
}  // namespace coup
