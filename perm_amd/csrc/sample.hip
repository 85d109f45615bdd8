// The next token of every row of logits (gfx950).
//
// With temperature T > 0 a token of logit x has the weight w = e^((x - max) / T). Tokens are ordered
// by falling logit, equal ones by rising number, and what is kept is a front of that order:
//
//     top_k   the first k tokens
//     top_p   of those, the ones before which less than top_p of their sum of weights lies
//     min_p   of those, the ones with w >= min_p
//
// (the first token always). Of the kept tokens, in the order of their numbers, the row's token is the
// first at which the sum of weights passes u times the whole of it. T <= 0: the first in the
// order. A NaN counts as minus infinity, which is never a token; a row of nothing else gives -1.
//
// Which token u falls on must not hang on the order in which weights are added: a vocabulary of 2^17
// tokens has borders 2^-17 apart, float32 sums err by 2^-20 of the whole. A weight is the whole
// number round(w 2^s), computed in float64, s = 62 - log2(vocabulary) up to 51, and sums are exact in 64 bits.
//
// A row is read two to four times, out of the caches but for the first, as a border has to be known before what it
// leaves can be summed. 256 rows of 151936 bfloat16 with settings of their own (78 MB): range 18.5 us, weigh 30
// (float64, the VALU two-thirds busy), collect 17, kept 16, and 26 in three launches of a workgroup a row. One row with
// top_k: five launches, 18.6 us, each as long as its latencies.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lowbit.h"

namespace cp {

constexpr int kBins = 2048;    // of a histogram
constexpr int kList = 2048;    // tokens that are sorted at most: two a thread
constexpr int kFew = 1024;     // tokens of a workgroup's lists, and ahead of the border that are listed
constexpr int kChunks = 1024;  // pieces of a row whose weights are summed by themselves, at most
constexpr int kChunkUnits = 256;  // of 16 bytes in a piece, at least
constexpr int kSplits = 64;     // workgroups of a row at most
constexpr int kFrontMost = 1024;  // top_k that several workgroups share
constexpr int kPeaks = 8;       // of a thread
constexpr int kMostPeaks = 4096;  // of a row
constexpr float kDead = -__builtin_inff();

struct SampleArgs {
  const void* logits;  // [rows], `step` elements apart
  int64_t step;
  int rows, vocab, shift;  // shift: the weights' s
  const void* u;       // [rows] float32, or float64
  int u64;
  const float *temperature, *top_p, *min_p;  // [rows], or null: the number
  const int* top_k;
  double t, p, m;
  int k;
  int* token;          // [rows]
  struct RowWork* work;  // [rows]
  uint32_t* peaks;       // [rows][splits][peaks_each]: largest keys of parts of the row
  int peaks_each;        // 64 .. 2048, a power of two
  int splits;          // workgroups of a row, where it is read by several
  int chunk_units, chunks, per;  // units of a chunk, chunks of a row and of a workgroup
};

// Order-preserving whole numbers of float32 (larger ones first do not: -0 is made 0 by the reader).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ (uint32_t)((int)b >> 31 | (int)0x80000000);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Place of a token in the order: larger comes first.
__device__ __forceinline__ uint64_t place(uint32_t key, int i) { return (uint64_t)key << 32 | (0xFFFFFFFFu - (uint32_t)i); }
__device__ __forceinline__ int token_of(uint64_t place) { return (int)(0xFFFFFFFFu - (uint32_t)place); }

__device__ __forceinline__ double fma_to(double a, double b, double c) {  // a b + c with c left as it is
  double y;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "s"(c));
  return y;
}

// round(2^s e^((x - max) / T)) with scale = log2 e / T: 2^n p(f), where p is the polynomial of degree 10 whose
// largest relative distance from 2^f over |f| <= 1/2 is least, 2.2e-16 (found by exchange). Numbers round as
// 1.5 x 2^52 (n) and 2^52 (the weight) are added, and lie in the low bits then. NaN and minus infinity weigh 0: fmax
// leaves the other. The largest logit is finite here.
struct Weigh {
  double top, scale;
  int shift;  // s
  __device__ __forceinline__ Weigh(float largest, double t, int s)
      : top(largest), scale(1.4426950408889634074 / t), shift(s) {}
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const double r = fmax(((double)x - top) * scale, -64.0);
    const double big = r + 6755399441055744.0, f = r - (big - 6755399441055744.0);
    double y = fma_to(7.037270609916633e-09, f, 1.0208537624759209e-07);
    y = fma_to(y, f, 1.321566288002748e-06);
    y = fma_to(y, f, 1.5252658118053735e-05);
    y = fma_to(y, f, 0.00015403529961050233);
    y = fma_to(y, f, 0.0013333558228558876);
    y = fma_to(y, f, 0.009618129108034647);
    y = fma_to(y, f, 0.05550410866445885);
    y = fma_to(y, f, 0.24022650695908768);
    y = fma_to(y, f, 0.6931471805599497);
    y = __builtin_fma(y, f, 1.0);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, big) + shift;
    const uint64_t b = __builtin_bit_cast(uint64_t, y);
    const double w = __builtin_bit_cast(double, ((uint64_t)((uint32_t)(b >> 32) + (n << 20)) << 32) | (uint32_t)b) +
                     4503599627370496.0;
    return __builtin_bit_cast(uint64_t, w) & 0xFFFFFFFFFFFFFull;
  }
  // Of any logit, also where the largest is an infinity.
  __device__ __forceinline__ uint64_t any(float x) const {
    return (double)x == top ? (uint64_t)1 << shift : (*this)(x);
  }
};

// One row's elements, 16 bytes a thread and step.
template <int DT>
struct RowReader {
  typedef typename Elem<DT>::T T;
  static constexpr int E = 16 / sizeof(T);
  const T* p;
  int vocab, off, units;  // off: elements of the first unit before the row
  __device__ __forceinline__ RowReader(const SampleArgs& a, int row) {
    p = (const T*)a.logits + (int64_t)row * a.step;
    vocab = a.vocab;
    off = (int)(reinterpret_cast<uintptr_t>(p) / sizeof(T) % E);
    units = (vocab + off + E - 1) / E;
  }
  __device__ __forceinline__ u32x4 load(int unit) const {
    const int i0 = unit * E - off;
    if (i0 >= 0 && i0 + E <= vocab) return *reinterpret_cast<const u32x4*>(p + i0);
    T e[E];
#pragma unroll
    for (int j = 0; j < E; ++j) e[j] = i0 + j >= 0 && i0 + j < vocab ? p[i0 + j] : (T)kDead;
    return __builtin_bit_cast(u32x4, e);
  }
  // Element j of a unit as it stands, and with NaN as minus infinity, -0 as 0.
  static __device__ __forceinline__ float raw(const u32x4& w, int j) {
    if constexpr (DT == CP_F32) {
      const uint32_t b = w[j];
      return __uint_as_float(b);
    } else {
      const uint32_t b = w[j >> 1];
      if constexpr (DT == CP_BF16)
        return __uint_as_float(j & 1 ? b & 0xFFFF0000u : b << 16);
      else
        return (float)__builtin_bit_cast(f16x2, b)[j & 1];
    }
  }
  static __device__ __forceinline__ float value(const u32x4& w, int j) { return fmaxf(raw(w, j), kDead) + 0.0f; }
  // f(unit, its 16 bytes, which of four) for the units first, first + by, ... before `end`; four loads in flight.
  template <class F>
  __device__ __forceinline__ void each(int first, int by, int end, F f) const {
    constexpr int U = 4;
    for (int g = first; g < end; g += U * by) {
      u32x4 w[U];
#pragma unroll
      for (int x = 0; x < U; ++x)
        if (g + x * by < end) w[x] = load(g + x * by);
#pragma unroll
      for (int x = 0; x < U; ++x)
        if (g + x * by < end) f(g + x * by, w[x], x);
    }
  }
};

// What the launches of a call hand on about a row.
struct RowWork {
  uint64_t mass[kBins];
  uint64_t list[kList + kFew];  // tokens among which the border is; top_p: and the ones ahead of them
  uint64_t chunk[kChunks];
  uint64_t first[kSplits];   // of every workgroup: its largest place,
  uint32_t top[kSplits], least[kSplits];  // its largest key, its least key's complement
  uint64_t before, goal;     // weight ahead of the border's bin, and the border's
  uint64_t cut;              // place of the last token kept
  uint32_t least_kept;       // key of the least logit that min_p leaves
  uint32_t n, ahead;         // tokens on either list, or that there were for it
  uint32_t from, to;         // keys of the border's list
  uint32_t done, whole;      // the row has its token; it is left to one workgroup
};

// How a row is dealt with.
enum RowKind { kGreedy, kWhole, kFront, kShare, kAll };

struct RowSettings {
  double t, p, m, u;
  uint64_t k;
  RowKind kind;
};

__device__ __forceinline__ RowSettings settings(const SampleArgs& a, int r) {
  RowSettings s;
  s.t = a.temperature ? (double)a.temperature[r] : a.t;
  if (s.t > 0.0) s.t = fmax(s.t, 1e-290);  // 1 / T stays finite; logits 2^-149 apart already weigh 0 there
  s.p = a.top_p ? (double)a.top_p[r] : a.p;
  const double m = a.min_p ? (double)a.min_p[r] : a.m;
  s.m = m > 0.0 ? fmin(m, 1.0) : 0.0;
  s.u = a.u64 ? ((const double*)a.u)[r] : (double)((const float*)a.u)[r];
  const int k = max(a.top_k ? a.top_k[r] : a.k, 0);
  s.k = k >= a.vocab ? 0 : k;
  s.kind = !(s.t > 0.0) ? kGreedy : s.k > kFrontMost ? kWhole : s.k ? kFront : s.p < 1.0 ? kShare : kAll;
  return s;
}

// Least whole number that is no less than p times the sum, and at least 1: the first token stays.
__device__ __forceinline__ uint64_t mass_goal(double p, uint64_t total) {
  const double g = ceil(fmax(p, 0.0) * (double)total);
  return g >= (double)total ? total : max((uint64_t)g, (uint64_t)1);
}
__device__ __forceinline__ uint64_t pick_goal(double u, uint64_t total) {
  const double g = floor(fmax(u, 0.0) * (double)total);
  return g >= (double)(total - 1) ? total - 1 : (uint64_t)g;
}

__device__ __forceinline__ uint64_t join64(int lo, int hi) { return (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo; }
// The value of lane ^ S, without LDS: within rows of 16 lanes by moves, beyond by swapping rows of two copies.
template <int S>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (S == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);   // within four: 1 0 3 2
  if constexpr (S == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);   // 2 3 0 1
  if constexpr (S == 4)  // eight in reverse, then each four of them
    return __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true), 0x1B, 0xF, 0xF, true);
  if constexpr (S == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, true);  // sixteen turned by eight
  if constexpr (S == 16) {
    const auto w = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? w[0] : w[1];
  } else {
    const auto w = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? w[0] : w[1];
  }
}
template <int S>
__device__ __forceinline__ uint64_t lane_xor64(uint64_t v) {
  return (uint64_t)lane_xor<S>((uint32_t)(v >> 32)) << 32 | lane_xor<S>((uint32_t)v);
}
// v put together over the wave, in every lane.
template <class F>
__device__ __forceinline__ uint64_t wave_all64(uint64_t v, F f) {
  v = f(v, lane_xor64<1>(v));
  v = f(v, lane_xor64<2>(v));
  v = f(v, lane_xor64<4>(v));
  v = f(v, lane_xor64<8>(v));
  v = f(v, lane_xor64<16>(v));
  return f(v, lane_xor64<32>(v));
}
// v of another lane by a move CTRL, 0 for lanes without one and in rows of 16 that ROWS leaves out.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lane_move64(uint64_t v) {
  return join64(__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false),
                __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false));
}
// Sum of v over the lanes up to this one: rows of 16 moved up by 1, 2, 4 and 8, then the last lanes of rows.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  v += lane_move64<0x111, 0xF>(v);
  v += lane_move64<0x112, 0xF>(v);
  v += lane_move64<0x114, 0xF>(v);
  v += lane_move64<0x118, 0xF>(v);
  v += lane_move64<0x142, 0xA>(v);
  return v + lane_move64<0x143, 0xC>(v);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
  return wave_all64(v, [](uint64_t a, uint64_t b) { return a + b; });
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  return wave_all64(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}

// The value of one lane, the same number in all.
__device__ __forceinline__ uint64_t read_lane64(uint64_t v, int lane) {
  return join64(__builtin_amdgcn_readlane((int)(uint32_t)v, lane), __builtin_amdgcn_readlane((int)(v >> 32), lane));
}

// Sum of v over the threads before this one, and over all W waves.
template <int W>
__device__ __forceinline__ uint64_t scan_block(uint64_t v, uint64_t* red, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t sum = wave_scan64(v);
  if (lane == 63) red[wave] = sum;
  __syncthreads();
  // the waves' sums in the first lanes of each row of 16 (by every thread for itself: 16 reads and 96 more operations)
  const int at = lane & 15;
  uint64_t s = at < W ? red[at] : 0;
  s += lane_move64<0x111, 0xF>(s);
  s += lane_move64<0x112, 0xF>(s);
  if (W > 4) {
    s += lane_move64<0x114, 0xF>(s);
    s += lane_move64<0x118, 0xF>(s);
  }
  const int w = __builtin_amdgcn_readfirstlane(wave);
  const uint64_t base = w ? read_lane64(s, w - 1) : 0;
  __syncthreads();
  *total = read_lane64(s, W - 1);
  return base + sum - v;
}

template <int W>
__device__ __forceinline__ uint64_t max_block(uint64_t v, uint64_t* red) {
  v = wave_max64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) v = red[w] > v ? red[w] : v;
  __syncthreads();
  return v;
}

// A step of a sort: values number t + 1024 e against partners o, j apart, in runs of k that fall and rise in turn.
template <int E>
__device__ __forceinline__ void sort_keep(uint64_t (&v)[E], const uint64_t (&o)[E], int t, int j, int k) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool first = !(t & j), down = !((t + 1024 * e) & k);  // down: the larger one first
    v[e] = (first == down) == (v[e] > o[e]) ? v[e] : o[e];
  }
}
template <int J, int E>
__device__ __forceinline__ void sort_step(uint64_t (&v)[E], int t, int k) {
  uint64_t o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = lane_xor64<J>(v[e]);
  sort_keep<E>(v, o, t, J, k);
}

// The 64 values of a wave, sorted, the largest first.
__device__ __forceinline__ void sort_lanes(uint64_t (&v)[1]) {
  const int t = threadIdx.x & 63;
  for (int k = 2; k <= 64; k <<= 1) {
    if (k > 32) sort_step<32>(v, t, k);
    if (k > 16) sort_step<16>(v, t, k);
    if (k > 8) sort_step<8>(v, t, k);
    if (k > 4) sort_step<4>(v, t, k);
    if (k > 2) sort_step<2>(v, t, k);
    sort_step<1>(v, t, k);
  }
}

// Up to 1024 E values, number t + 1024 e in thread t's v[e], sorted, the largest first (threads past the n
// of them hold 0): a bitonic sort, whose steps within a wave need no LDS.
template <int E>
__device__ __forceinline__ void sort_block(uint64_t (&v)[E], int n, uint64_t* list) {
  const int t = threadIdx.x;
  int size = 64;
  while (size < n) size <<= 1;
  for (int k = 2; k <= size; k <<= 1) {
    int j = k >> 1;
    if (E > 1 && j == 1024) {
      const uint64_t a = v[0], b = v[E - 1];
      v[0] = a > b ? a : b, v[E - 1] = a > b ? b : a;
      j >>= 1;
    }
    for (; j >= 64; j >>= 1) {
      uint64_t o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) list[t + 1024 * e] = v[e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = list[(t ^ j) + 1024 * e];
      __syncthreads();
      sort_keep<E>(v, o, t, j, k);
    }
    if (j >= 32) sort_step<32>(v, t, k);
    if (j >= 16) sort_step<16>(v, t, k);
    if (j >= 8) sort_step<8>(v, t, k);
    if (j >= 4) sort_step<4>(v, t, k);
    if (j >= 2) sort_step<2>(v, t, k);
    sort_step<1>(v, t, k);
  }
}

// Bins of falling logits, as many as bring the least logit, or the one from which on weights are 0, to the
// last of them. Monotone, as subtraction, product and conversion round monotonically; where the
// largest is an infinity, the others' differences or their products with 0 go to the last bin.
struct Bins {
  float top, per;
  __device__ __forceinline__ Bins() {}
  __device__ __forceinline__ Bins(float largest, float least, int shift, double t) : top(largest) {
    const double span = fmin((double)largest - (double)least, (shift + 2) * 0.6931471805599453 * t);
    per = span > 0.0 ? (float)fmin((double)kBins / span, 3e38) : 0.0f;
    if (!(per > 0.0f)) per = 0.0f;
  }
  __device__ __forceinline__ int operator()(float x) const { return x == top ? 0 : finite(x); }
  // The same where the largest is finite.
  __device__ __forceinline__ int finite(float x) const { return min((int)fminf((top - x) * per, 4e6f), kBins - 1); }
};

// The least key in (lo, hi] of which `enough` holds, as it does of hi and of all above one it holds of. A wave
// tries 64 at a time.
template <class F>
__device__ __forceinline__ uint32_t least_key(uint32_t lo, uint32_t hi, F enough) {
  const uint32_t lane = threadIdx.x & 63;
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + 63) / 64, mine = hi - lo > step * (lane + 1) ? lo + step * (lane + 1) : hi;
    const int at = __ffsll((unsigned long long)__ballot(enough(mine))) - 1;
    const uint32_t end = hi - lo > step * (at + 1) ? lo + step * (at + 1) : hi;
    lo += step * at;
    hi = end;
  }
  return __builtin_amdgcn_readfirstlane(hi);
}
constexpr uint32_t kDeadKey = 0x007FFFFFu;  // of minus infinity

// The least weight that min_p leaves: the largest logit's is one.
__device__ __forceinline__ double least_weight(const Weigh& weigh, double m) {
  return ceil(m * (double)((uint64_t)1 << weigh.shift));
}

// The least key whose weight is one.
__device__ __forceinline__ uint32_t least_kept(const Weigh& weigh, float top, double m) {
  if (!(m > 0.0)) return kDeadKey + 1;
  const double least = least_weight(weigh, m);
  return least_key(kDeadKey, key_of(top),
                   [&](uint32_t k) { return k == key_of(top) || (double)weigh(value_of(k)) >= least; });
}

struct SampleShared {
  uint64_t mass[kBins];  // of a histogram
  uint64_t chunk[kChunks];
  uint64_t list[kList];
  uint64_t red[16];
  uint32_t count[kBins];
  uint32_t n;
  uint64_t pick[4];
};

// Number `at` of the n tokens of the list in LDS, sorted, into sm.pick[3].
template <int E>
__device__ __forceinline__ void pick_sorted(SampleShared& sm, int n, int at) {
  const int t = threadIdx.x;
  uint64_t v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = t + 1024 * e < n ? sm.list[t + 1024 * e] : 0;
  __syncthreads();
  sort_block<E>(v, n, sm.list);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (t + 1024 * e == at) sm.pick[3] = v[e];
}

// The place of the last token kept among the n of the list in LDS: the one before which, `before` included,
// less than goal lies.
template <int E>
__device__ __forceinline__ uint64_t last_kept(SampleShared& sm, const Weigh& weigh, int n, uint64_t before,
                                              uint64_t goal) {
  const int t = threadIdx.x;
  uint64_t v[E], sum, least = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = t + 1024 * e < n ? sm.list[t + 1024 * e] : 0;
  __syncthreads();
  sort_block<E>(v, n, sm.list);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint64_t w = t + 1024 * e < n ? weigh.any(value_of((uint32_t)(v[e] >> 32))) : 0;
    const uint64_t b = before + scan_block<16>(w, sm.red, &sum);
    before += sum;
    if (t + 1024 * e < n && b < goal && ~v[e] > least) least = ~v[e];
  }
  return ~max_block<16>(least, sm.red);
}

// The token at which u falls among those of places v and weights w (0: not kept), in the order of numbers:
// weights by bins of numbers, then the border's bin, of a 2048th of the vocabulary.
template <int E>
__device__ __forceinline__ int by_number(SampleShared& sm, const uint64_t (&v)[E], const uint64_t (&w)[E], double u, int vocab) {
  const int t = threadIdx.x;
  for (int i = t; i < kBins; i += 1024) sm.mass[i] = 0;
  if (t == 0) sm.n = 0;
  __syncthreads();
  int bin[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    bin[e] = (int)((int64_t)token_of(v[e]) * kBins / vocab);
    if (w[e]) atomicAdd((unsigned long long*)&sm.mass[bin[e]], (unsigned long long)w[e]);
  }
  __syncthreads();
  uint64_t kept;
  const uint64_t m0 = sm.mass[2 * t], m1 = sm.mass[2 * t + 1], b = scan_block<16>(m0 + m1, sm.red, &kept);
  const uint64_t pick = pick_goal(u, kept);
  if (b <= pick && b + m0 > pick) sm.pick[0] = 2 * t, sm.pick[1] = b;
  else if (b + m0 <= pick && b + m0 + m1 > pick) sm.pick[0] = 2 * t + 1, sm.pick[1] = b + m0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (w[e] && bin[e] == (int)sm.pick[0]) {
      const uint32_t at = atomicAdd(&sm.n, 1u);
      sm.list[at] = (uint32_t)v[e];  // larger for smaller numbers
      sm.mass[at] = w[e];
    }
  __syncthreads();
  for (int i = t; i < (int)sm.n; i += 1024) {
    uint64_t before = sm.pick[1];
    for (int j = 0; j < (int)sm.n; ++j) before += sm.list[j] > sm.list[i] ? sm.mass[j] : 0;
    if (before <= pick && before + sm.mass[i] > pick) sm.pick[2] = 0xFFFFFFFFu - (uint32_t)sm.list[i];
  }
  __syncthreads();
  return (int)sm.pick[2];
}

__device__ __forceinline__ uint64_t lane_value64(uint64_t v, int lane) {
  return join64(__shfl((int)(uint32_t)v, lane), __shfl((int)(v >> 32), lane));
}

// choose() of up to 64 tokens, by one wave: two sorts and three sums in registers (a launch of one row 8 us as choose
// does it, 4.3 so).
__device__ __forceinline__ int choose_few(const uint64_t* list, const Weigh& weigh, int n, const RowSettings& s, uint64_t goal) {
  const int lane = threadIdx.x & 63;
  const double least = least_weight(weigh, s.m);
  uint64_t v[1] = {lane < n ? list[lane] : 0};
  sort_lanes(v);
  const int last = s.k ? min(n, (int)min(s.k, (uint64_t)64)) : n;
  uint64_t w = lane < last ? weigh.any(value_of((uint32_t)(v[0] >> 32))) : 0;
  uint64_t sum = wave_scan64(w);
  const uint64_t total = lane_value64(sum, 63), share = goal ? goal : s.p < 1.0 ? mass_goal(s.p, total) : total;
  const bool keep = lane < last && (lane == 0 || (sum - w < share && (double)w >= least));
  w = keep ? w : 0;
  const uint64_t pick = pick_goal(s.u, lane_value64(wave_scan64(w), 63));
  uint64_t by[1] = {keep ? (uint64_t)(uint32_t)v[0] << 32 | (uint32_t)lane : 0};  // by rising number, the kept ones first
  sort_lanes(by);
  const uint64_t own = lane_value64(w, (int)(by[0] & 63)), mine = by[0] ? own : 0;
  sum = wave_scan64(mine);
  const unsigned long long hit = __ballot(sum > pick && sum - mine <= pick);
  return token_of((uint64_t)(uint32_t)__shfl((int)(by[0] >> 32), __ffsll(hit) - 1));
}

// The bin, of values x0 in bin 2 t and x1 in the next, in which their sum reaches goal, and the sum before it.
__device__ __forceinline__ int border_bin(SampleShared& sm, uint64_t x0, uint64_t x1, uint64_t b, uint64_t goal, uint64_t* before) {
  const int t = threadIdx.x;
  if (b < goal && b + x0 >= goal) sm.pick[0] = 2 * t, sm.pick[1] = b;
  else if (b + x0 < goal && b + x0 + x1 >= goal) sm.pick[0] = 2 * t + 1, sm.pick[1] = b + x0;
  __syncthreads();
  *before = sm.pick[1];
  return (int)sm.pick[0];
}

// The values v in bin `border` of theirs (at) onto the list, side by side: how many.
__device__ __forceinline__ int gather(SampleShared& sm, const uint64_t (&v)[2], const int (&at)[2], int border) {
  if (threadIdx.x == 0) sm.n = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (at[e] == border) sm.list[atomicAdd(&sm.n, 1u)] = v[e];
  __syncthreads();
  return (int)sm.n;
}

// The place of the last token kept among those of places v, weights w and bins at, and its bin: the one before which,
// `before` included, less than goal lies (goal 0: the share p of their sum). A histogram finds the bin, and its
// tokens alone are sorted: by one wave where they are up to 64. sm.mass is 0 on entry.
__device__ __forceinline__ uint64_t last_by_mass(SampleShared& sm, const Weigh& weigh, const uint64_t (&v)[2], const uint64_t (&w)[2],
                                                 const int (&at)[2], uint64_t before, uint64_t goal, double p, int* border) {
  const int t = threadIdx.x, lane = t & 63;
  uint64_t sum;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (w[e]) atomicAdd((unsigned long long*)&sm.mass[at[e]], (unsigned long long)w[e]);
  __syncthreads();
  const uint64_t m0 = sm.mass[2 * t], m1 = sm.mass[2 * t + 1], b = before + scan_block<16>(m0 + m1, sm.red, &sum);
  const uint64_t share = goal ? goal : mass_goal(p, sum);
  *border = border_bin(sm, m0, m1, b, share, &before);
  const int m = gather(sm, v, at, *border);
  if (m > 1024) return last_kept<2>(sm, weigh, m, before, share);
  if (m > 64) return last_kept<1>(sm, weigh, m, before, share);
  if (t < 64) {
    uint64_t x[1] = {lane < m ? sm.list[lane] : 0};
    sort_lanes(x);
    const uint64_t y = lane < m ? weigh.any(value_of((uint32_t)(x[0] >> 32))) : 0;
    const uint64_t sum = wave_scan64(y);
    const unsigned long long kept = __ballot(lane < m && before + sum - y < share);  // a front of the lanes
    if (lane == __popcll(kept) - 1) sm.pick[3] = x[0];
  }
  __syncthreads();
  return sm.pick[3];
}

// Chooses among the n tokens of the list in LDS, all that may be kept: k, p, m and u as in the file's heading (k 0:
// all n). goal: top_p's, where the list is not all the weight there is (0: it is). Each border is found by a
// histogram of the list over `bin`, and the tokens of its bin alone are sorted (1100 tokens sorted as a whole 21 us a
// row, so 13).
__device__ __forceinline__ int choose(SampleShared& sm, const Weigh& weigh, const Bins& bin, int n, const RowSettings& s,
                                      uint64_t goal, int vocab) {
  const int t = threadIdx.x, lane = t & 63;
  const double least = least_weight(weigh, s.m);
  uint64_t v[2], w[2], sum, before;
  int at[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    v[e] = t + 1024 * e < n ? sm.list[t + 1024 * e] : 0;
    at[e] = v[e] ? bin(value_of((uint32_t)(v[e] >> 32))) : kBins;
    sm.count[t + 1024 * e] = 0;
    sm.mass[t + 1024 * e] = 0;
  }
  auto drop = [&](int border, uint64_t cut) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (at[e] > border || (at[e] == border && v[e] < cut)) v[e] = 0, at[e] = kBins;
  };
  __syncthreads();
  if (s.k && (uint64_t)n > s.k) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (v[e]) atomicAdd(&sm.count[at[e]], 1u);
    __syncthreads();
    const uint64_t c0 = sm.count[2 * t], c1 = sm.count[2 * t + 1], b = scan_block<16>(c0 + c1, sm.red, &sum);
    const int border = border_bin(sm, c0, c1, b, s.k, &before);
    const int m = gather(sm, v, at, border), need = (int)(s.k - before);  // of m
    if (m <= 64) {
      if (t < 64) {
        uint64_t x[1] = {lane < m ? sm.list[lane] : 0};
        sort_lanes(x);
        if (lane == need - 1) sm.pick[3] = x[0];
      }
    } else if (m <= 1024) {
      pick_sorted<1>(sm, m, need - 1);
    } else {
      pick_sorted<2>(sm, m, need - 1);
    }
    __syncthreads();
    drop(border, sm.pick[3]);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) w[e] = v[e] ? weigh.any(value_of((uint32_t)(v[e] >> 32))) : 0;
  if (goal || s.p < 1.0) {
    int border;
    const uint64_t cut = last_by_mass(sm, weigh, v, w, at, 0, goal, s.p, &border);
    drop(border, cut);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) w[e] = v[e] && (double)w[e] >= least ? w[e] : 0;
  __syncthreads();
  return by_number<2>(sm, v, w, s.u, vocab);
}

// The sum of value(i, x) over chunk c, by one wave.
template <int DT, class F>
__device__ __forceinline__ uint64_t chunk_sum(const SampleArgs& a, const RowReader<DT>& row, int c, F value) {
  const int lane = threadIdx.x & 63, g0 = c * a.chunk_units, g1 = min(row.units, g0 + a.chunk_units);
  uint64_t v = 0;
  for (int g = g0 + lane; g < g1; g += 256) {
    u32x4 w[4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (g + 64 * x < g1) w[x] = row.load(g + 64 * x);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (g + 64 * x < g1) {
#pragma unroll
        for (int j = 0; j < RowReader<DT>::E; ++j)
          v += value((g + 64 * x) * RowReader<DT>::E - row.off + j, RowReader<DT>::raw(w[x], j));
      }
  }
  return wave_sum64(v);
}

// The weights of chunk c's logits from `from` on, by one wave. A lane weighs only those of its own that are: four
// units lie in LDS (own, 16 bytes a thread and unit, 256 threads apart), from which it takes them one by one,
// so that a step of a wave costs what its fullest lane has. 256 rows of which a ninth is kept: all
// weighed 43 us, so 30.
template <int DT>
__device__ __forceinline__ uint64_t chunk_sum_from(const SampleArgs& a, const RowReader<DT>& row, int c, const Weigh& weigh,
                                                   float from, u32x4* own) {
  typedef typename Elem<DT>::T T;
  constexpr int E = RowReader<DT>::E;
  const int lane = threadIdx.x & 63, g0 = c * a.chunk_units, g1 = min(row.units, g0 + a.chunk_units);
  uint64_t v = 0;
  for (int g = g0 + lane; g < g1; g += 256) {
    uint32_t mine = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (g + 64 * x >= g1) break;
      const u32x4 w = row.load(g + 64 * x);
      own[256 * x] = w;
#pragma unroll
      for (int j = 0; j < E; ++j) mine |= (RowReader<DT>::raw(w, j) >= from ? 1u : 0u) << (E * x + j);
    }
    while (mine) {
      const int i = __ffs(mine) - 1;
      mine &= mine - 1;
      v += weigh((float)reinterpret_cast<const T*>(own + 256 * (i / E))[i % E]);
    }
  }
  return wave_sum64(v);
}

// The number of the first token at which the sum of value(i, x) in the order of numbers passes goal, which
// is less than the whole. The chunks' sums are in LDS. 1024 threads.
template <int DT, class F>
__device__ __forceinline__ int find(const SampleArgs& a, SampleShared& sm, const RowReader<DT>& row, uint64_t goal,
                                    F value) {
  constexpr int E = RowReader<DT>::E;
  uint64_t sum;
  const uint64_t mine = (int)threadIdx.x < a.chunks ? sm.chunk[threadIdx.x] : 0;
  const uint64_t before = scan_block<16>(mine, sm.red, &sum);
  if (before <= goal && before + mine > goal) sm.pick[0] = threadIdx.x, sm.pick[1] = before;
  __syncthreads();
  const int c = (int)sm.pick[0], g1 = min(row.units, (c + 1) * a.chunk_units);
  uint64_t base = sm.pick[1];
  for (int g0 = c * a.chunk_units; g0 < g1 && base <= goal; g0 += 1024) {
    const int g = g0 + threadIdx.x;
    uint64_t v[E], all = 0;
    if (g < g1) {
      const u32x4 w = row.load(g);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        v[j] = value(g * E - row.off + j, RowReader<DT>::raw(w, j));
        all += v[j];
      }
    }
    uint64_t b = base + scan_block<16>(all, sm.red, &sum);
    if (b <= goal && b + all > goal) {
      int j = 0;
#pragma unroll
      for (int x = 0; x < E; ++x) {
        b += v[x];
        if (b <= goal) j = x + 1;
      }
      sm.pick[2] = (uint64_t)(g * E - row.off + min(j, E - 1));
    }
    base += sum;
  }
  __syncthreads();
  return (int)sm.pick[2];
}

template <int DT>
struct Sampler {
  const SampleArgs& a;
  SampleShared& sm;
  RowReader<DT> row;
  Weigh weigh;
  Bins bin;

  static constexpr int E = RowReader<DT>::E;

  template <class F>
  __device__ __forceinline__ void tokens(F f) const {
    row.each(threadIdx.x, 1024, row.units, [&](int unit, const u32x4& w, int) {
      const int i0 = unit * E - row.off;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float x = RowReader<DT>::value(w, j);
        if (x != kDead) f(i0 + j, x);
      }
    });
  }

  __device__ __forceinline__ void clear_bins() {
    __syncthreads();  // every wave has read what it needs of the last histogram
    for (int i = threadIdx.x; i < kBins; i += 1024) sm.mass[i] = 0, sm.count[i] = 0;
    __syncthreads();
  }

  // The border's bin in the histogram: the first at whose end `by_count` tokens or `by_mass` of weight
  // are reached (whichever is not 0), its number in *at, tokens and weight before it.
  __device__ __forceinline__ void border(uint64_t by_count, uint64_t by_mass, int* at, uint64_t* count, uint64_t* mass) {
    const int i = 2 * threadIdx.x;
    uint64_t all;
    const uint64_t c0 = sm.count[i], c1 = sm.count[i + 1], m0 = sm.mass[i], m1 = sm.mass[i + 1];
    const uint64_t c = scan_block<16>(c0 + c1, sm.red, &all), m = scan_block<16>(m0 + m1, sm.red, &all);
    if (threadIdx.x == 0) sm.pick[0] = kBins - 1, sm.pick[1] = sm.pick[2] = 0;
    __syncthreads();
    const uint64_t goal = by_count ? by_count : by_mass;
    const uint64_t b = by_count ? c : m, x0 = by_count ? c0 : m0, x1 = by_count ? c1 : m1;
    if (b < goal && b + x0 >= goal) sm.pick[0] = i, sm.pick[1] = c, sm.pick[2] = m;
    else if (b + x0 < goal && b + x0 + x1 >= goal) sm.pick[0] = i + 1, sm.pick[1] = c + c0, sm.pick[2] = m + m0;
    __syncthreads();
    *at = (int)sm.pick[0], *count = sm.pick[1], *mass = sm.pick[2];
    __syncthreads();
  }

  // Tokens with lo <= key <= hi into the list; false where they are too many.
  __device__ __forceinline__ bool collect(uint32_t lo, uint32_t hi, uint64_t cut, int* n) {
    if (threadIdx.x == 0) sm.n = 0;
    __syncthreads();
    tokens([&](int i, float x) {
      const uint32_t k = key_of(x);
      if (k >= lo && k <= hi && place(k, i) >= cut) {
        const uint32_t at = atomicAdd(&sm.n, 1u);
        if (at < kList) sm.list[at] = place(k, i);
      }
    });
    __syncthreads();
    *n = (int)min(sm.n, 0x7FFFFFFFu);
    const bool fits = sm.n <= kList;
    __syncthreads();
    return fits;
  }

  // The least key of a bin: keys rise as bins fall.
  __device__ __forceinline__ uint32_t bin_start(int b) const {
    uint32_t lo = key_of(kDead) + 1, hi = key_of(bin.top);  // bin(hi) = 0 <= b
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (bin(value_of(mid)) <= b) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }

  // Of the tokens at or above `cut`, the place of the last one kept: by_count tokens, or those before which
  // less than by_mass lies.
  //
  // A histogram finds the bin the border lies in; the bin's keys are split again until its tokens fit
  // the list, or are all equal.
  __device__ __forceinline__ uint64_t front(uint64_t cut, uint64_t by_count, uint64_t by_mass, int at, uint64_t count,
                                       uint64_t mass) {
    uint32_t hi = at == 0 ? key_of(bin.top) : bin_start(at - 1) - 1, lo = bin_start(at);
    for (;;) {
      int n;
      const uint64_t in_bin = sm.count[at];
      if (in_bin <= kList) {
        collect(lo, hi, cut, &n);
        if (by_count) {
          pick_sorted<2>(sm, n, (int)(by_count - count) - 1);
          __syncthreads();
          return sm.pick[3];
        }
        return last_kept<2>(sm, weigh, n, mass, by_mass);
      }
      if (lo == hi) break;
      const int s = max(0, 32 - __clz(hi - lo) - 11);
      clear_bins();
      const uint32_t top_key = hi;
      tokens([&](int i, float x) {
        const uint32_t k = key_of(x);
        if (k >= lo && k <= top_key && place(k, i) >= cut) {
          const uint32_t b = (top_key - k) >> s;
          atomicAdd(&sm.count[b], 1u);
          if (by_mass) atomicAdd((unsigned long long*)&sm.mass[b], (unsigned long long)weigh.any(x));
        }
      });
      __syncthreads();
      uint64_t c, m;
      border(by_count ? by_count - count : 0, by_count ? 0 : by_mass - mass, &at, &c, &m);
      count += c, mass += m;
      hi = top_key - ((uint32_t)at << s);
      lo = max(lo, hi - ((1u << s) - 1));
    }
    // equal logits: the first of them by number
    uint64_t need;
    if (by_count) {
      need = by_count - count;
    } else {
      const uint64_t w = weigh.any(value_of(hi));
      need = w ? (by_mass - mass + w - 1) / w : 1;
    }
    return nth(hi, cut, need);
  }

  // Sums value(i, x) over chunks of the row into sm.chunk, then finds the chunk in which the sum in the
  // order of numbers passes `goal`: the number of the first token at which it does.
  template <class F>
  __device__ __forceinline__ void chunk_sums(F value) {
    __syncthreads();
    for (int c = threadIdx.x >> 6; c < a.chunks; c += 16) {
      const uint64_t v = chunk_sum<DT>(a, row, c, value);
      if ((threadIdx.x & 63) == 0) sm.chunk[c] = v;
    }
    __syncthreads();
  }

  // The place of the need'th token with this key at or above `cut`, by number.
  __device__ __forceinline__ uint64_t nth(uint32_t key, uint64_t cut, uint64_t need) {
    auto one = [&](int i, float x) -> uint64_t { return x == value_of(key) && place(key, i) >= cut; };
    chunk_sums(one);
    uint64_t all;
    scan_block<16>((int)threadIdx.x < a.chunks ? sm.chunk[threadIdx.x] : 0, sm.red, &all);
    if (all == 0) return cut;  // no such token: not reached
    return place(key, find<DT>(a, sm, row, min(need, all) - 1, one));
  }

  // A row by one workgroup, whatever it holds.
  __device__ __forceinline__ int whole(const RowSettings& s) {
    uint64_t all, k = s.k, alive = 0, cut = 0, count, mass;
    int at;
    tokens([&](int, float) { ++alive; });
    scan_block<16>(alive, sm.red, &all);
    if (k >= all) k = 0;
    if (k) {
      clear_bins();
      tokens([&](int, float x) { atomicAdd(&sm.count[bin(x)], 1u); });
      __syncthreads();
      border(k, 0, &at, &count, &mass);
      cut = front(0, k, 0, at, count, 0);
    }
    if (s.p < 1.0) {
      clear_bins();
      tokens([&](int i, float x) {
        if (place(key_of(x), i) < cut) return;
        const int b = bin(x);
        atomicAdd(&sm.count[b], 1u);
        atomicAdd((unsigned long long*)&sm.mass[b], (unsigned long long)weigh.any(x));
      });
      __syncthreads();
      scan_block<16>(sm.mass[threadIdx.x] + sm.mass[threadIdx.x + 1024], sm.red, &all);
      const uint64_t goal = mass_goal(s.p, all);
      border(0, goal, &at, &count, &mass);
      cut = front(cut, 0, goal, at, count, mass);
    }
    const double least = s.m * (double)((uint64_t)1 << weigh.shift);
    auto value = [&](int i, float x) -> uint64_t {
      if (!(x > kDead) || place(key_of(x + 0.0f), i) < cut) return 0;
      const uint64_t w = weigh.any(x);
      return (double)w >= least ? w : 0;
    };
    chunk_sums(value);
    scan_block<16>((int)threadIdx.x < a.chunks ? sm.chunk[threadIdx.x] : 0, sm.red, &all);
    return find<DT>(a, sm, row, pick_goal(s.u, all), value);
  }
};

// A row's largest and least logit as its first launch left them (nothing but minus infinity: kDead).
struct RowRange {
  float top, least;
};
__device__ __forceinline__ RowRange row_range(const SampleArgs& a, const RowWork& w) {
  const int lane = threadIdx.x & 63;
  const uint64_t both = wave_all64(lane < a.splits ? (uint64_t)w.top[lane] << 32 | w.least[lane] : 0, [](uint64_t a, uint64_t b) {
    return (uint64_t)max((uint32_t)(a >> 32), (uint32_t)(b >> 32)) << 32 | max((uint32_t)a, (uint32_t)b);
  });
  const uint32_t top = __builtin_amdgcn_readfirstlane((uint32_t)(both >> 32)), least = __builtin_amdgcn_readfirstlane((uint32_t)both);
  return {top ? value_of(top) : kDead, value_of(~least)};
}

// Launch 1, a.splits workgroups a row as all others that read it: its largest logit (and the first token that
// has it, where that is the answer), its least, and what the next ones add to cleared. top_k: also the
// largest of every thread's loads, from which the next launch tells how far down to look.
template <int DT>
__global__ __launch_bounds__(256) void sample_range_kernel(SampleArgs a) {
  __shared__ uint64_t red[4];
  const int r = blockIdx.x / a.splits, at = blockIdx.x % a.splits;
  const RowSettings s = settings(a, r);
  const RowReader<DT> row(a, r);
  RowWork& w = a.work[r];
  const int g0 = at * a.per * a.chunk_units, g1 = min(row.units, (at + 1) * a.per * a.chunk_units);
  constexpr int E = RowReader<DT>::E;
  if (s.kind == kGreedy) {
    uint64_t best = 0;
    row.each(g0 + threadIdx.x, 256, g1, [&](int unit, const u32x4& v, int) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float x = RowReader<DT>::value(v, j);
        const uint64_t p = place(key_of(x), unit * E - row.off + j);
        best = x != kDead && p > best ? p : best;
      }
    });
    best = max_block<4>(best, red);
    if (threadIdx.x == 0) w.first[at] = best;
  } else {
    float peak[kPeaks], least = __builtin_inff();
#pragma unroll
    for (int i = 0; i < kPeaks; ++i) peak[i] = kDead;
    row.each(g0 + threadIdx.x, 256, g1, [&](int, const u32x4& v, int x) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float y = RowReader<DT>::raw(v, j);
        float& to = peak[2 * x + (j >= E / 2)];
        to = fmaxf(to, y);
        least = fminf(least, y == kDead ? __builtin_inff() : y);
      }
    });
    if (s.kind == kFront) {
      uint32_t* to = a.peaks + (int64_t)blockIdx.x * a.peaks_each;
      float p[kPeaks];
#pragma unroll
      for (int i = 0; i < kPeaks; ++i) p[i] = peak[i];
#pragma unroll
      for (int n = kPeaks / 2; n > 0; n >>= 1)
        if (a.peaks_each <= 256 * n) {
#pragma unroll
          for (int i = 0; i < n; ++i) p[i] = fmaxf(p[i], p[i + n]);
        }
      int stride = 1;  // threads that share a peak
      for (; a.peaks_each * stride < 256; stride *= 2) p[0] = fmaxf(p[0], __shfl_xor(p[0], stride));
#pragma unroll
      for (int i = 0; i < kPeaks; ++i)
        if ((i == 0 || 256 * i < a.peaks_each) && threadIdx.x % stride == 0)
          to[256 * i + threadIdx.x / stride] = p[i] == kDead ? 0 : key_of(p[i] + 0.0f);
    }
    float top = peak[0];
#pragma unroll
    for (int i = 1; i < kPeaks; ++i) top = fmaxf(top, peak[i]);
    const uint64_t hi = max_block<4>(top == kDead ? 0 : key_of(top + 0.0f), red);
    const uint64_t lo = max_block<4>((uint32_t)~key_of(least + 0.0f), red);
    if (threadIdx.x == 0) w.top[at] = (uint32_t)hi, w.least[at] = (uint32_t)lo;
    if (s.kind == kShare)
      for (int i = at * 256 + threadIdx.x; i < kBins; i += a.splits * 256) w.mass[i] = 0;
  }
  if (at == 0 && threadIdx.x == 0) w.n = w.ahead = w.done = w.whole = 0;
}

// Launch 2. top_k: a logit that k tokens reach, as k of the peaks do. top_p: the weight in each bin. Neither: the
// chunks' weights.
template <int DT>
__global__ __launch_bounds__(256) void sample_weigh_kernel(SampleArgs a) {
  __shared__ uint64_t mass[kBins];
  __shared__ uint64_t red[4];
  __shared__ uint32_t pick;
  const int r = blockIdx.x / a.splits, at = blockIdx.x % a.splits;
  const RowSettings s = settings(a, r);
  if (s.kind == kGreedy || s.kind == kWhole || (s.kind == kFront && at != r % a.splits)) return;  // on every XCD in turn
  RowWork& w = a.work[r];
  const RowRange range = row_range(a, w);
  if (!(fabsf(range.top) < __builtin_inff())) return;  // an infinity: one workgroup deals with it
  constexpr int N = kBins / 256;
  if (s.kind == kFront) {
    uint32_t* count = reinterpret_cast<uint32_t*>(mass);
    const uint32_t* peaks = a.peaks + (int64_t)r * a.splits * a.peaks_each;
    const int n = a.splits * a.peaks_each;  // at most kMostPeaks
    uint32_t mine[kMostPeaks / 256], low = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < kMostPeaks / 256; ++i) {
      const int at = threadIdx.x + 256 * i;
      mine[i] = at < n ? peaks[at] : 0;
    }
    for (int i = threadIdx.x; i < kBins; i += 256) count[i] = 0;
    if (threadIdx.x == 0) pick = kBins;
    // bins over the peaks alone
#pragma unroll
    for (int i = 0; i < kMostPeaks / 256; ++i) low = min(low, mine[i] ? mine[i] : 0xFFFFFFFFu);
    low = ~(uint32_t)max_block<4>((uint32_t)~low, red);
    const Bins bin(range.top, value_of(low), a.shift, __builtin_inf());
#pragma unroll
    for (int i = 0; i < kMostPeaks / 256; ++i)
      if (mine[i]) atomicAdd(&count[bin(value_of(mine[i]))], 1u);
    __syncthreads();
    uint64_t sum = 0, all;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += count[threadIdx.x * N + i];
    uint64_t before = scan_block<4>(sum, red, &all);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t c = count[threadIdx.x * N + i];
      if (before < s.k && before + c >= s.k) pick = threadIdx.x * N + i;
      before += c;
    }
    __syncthreads();
    const int border = (int)pick;
    // fewer peaks than top_k: every token may be kept
    const uint32_t from = border == kBins ? kDeadKey + 1
                                          : least_key(kDeadKey, key_of(range.top),
                                                      [&](uint32_t k) { return bin(value_of(k)) <= border; });
    if (threadIdx.x == 0) w.from = from, w.to = 0xFFFFFFFFu;
    return;
  }
  const RowReader<DT> row(a, r);
  const int c0 = at * a.per, c1 = min(a.chunks, c0 + a.per);
  constexpr int E = RowReader<DT>::E;
  const Weigh weigh(range.top, s.t, a.shift);
  if (s.kind == kAll) {
    const uint32_t least = least_kept(weigh, range.top, s.m);
    const float from = value_of(least);
    for (int c = c0 + (threadIdx.x >> 6); c < c1; c += 4) {
      const uint64_t v = chunk_sum<DT>(a, row, c, [&](int, float x) { return weigh(x >= from ? x : kDead); });
      if ((threadIdx.x & 63) == 0) w.chunk[c] = v;
    }
    if (at == 0 && threadIdx.x == 0) w.least_kept = least;
    return;
  }
  const int g0 = c0 * a.chunk_units, g1 = min(row.units, c1 * a.chunk_units);
  const Bins bin(range.top, range.least, a.shift, s.t);
  for (int i = threadIdx.x; i < kBins; i += 256) mass[i] = 0;
  __syncthreads();
  row.each(g0 + threadIdx.x, 256, g1, [&](int, const u32x4& v, int) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float x = RowReader<DT>::raw(v, j);
      const uint64_t y = weigh(x);
      if (y) atomicAdd((unsigned long long*)&mass[bin.finite(x)], (unsigned long long)y);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += 256)
    if (mass[i]) atomicAdd((unsigned long long*)&w.mass[i], (unsigned long long)mass[i]);
}

// Launch 3, a workgroup a row with top_p: the bin in which its border lies, that bin's keys, and min_p's. (The last
// workgroup of the launch before could do it, but the fence that it takes costs each of them an L2
// written back: 45 -> 303 us.)
__global__ __launch_bounds__(256) void sample_border_kernel(SampleArgs a) {
  __shared__ uint64_t red[4];
  __shared__ int pick;
  const int r = blockIdx.x;
  const RowSettings s = settings(a, r);
  if (s.kind != kShare) return;
  RowWork& w = a.work[r];
  const RowRange range = row_range(a, w);
  if (!(fabsf(range.top) < __builtin_inff())) return;
  constexpr int N = kBins / 256;
  uint64_t v[N], sum = 0, all;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = w.mass[threadIdx.x * N + i];
    sum += v[i];
  }
  uint64_t before = scan_block<4>(sum, red, &all);
  const uint64_t goal = mass_goal(s.p, all);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (before < goal && before + v[i] >= goal) pick = threadIdx.x * N + i, w.before = before;
    before += v[i];
  }
  __syncthreads();
  const int border = pick;
  const Bins bin(range.top, range.least, a.shift, s.t);
  // three searches, a wave each
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave == 0) {
    const uint32_t from = least_key(kDeadKey, key_of(range.top), [&](uint32_t k) { return bin(value_of(k)) <= border; });
    if (lane == 0) w.from = from, w.goal = goal;
  } else if (wave == 1) {
    const uint32_t to = border == 0 ? 0xFFFFFFFFu
                                    : least_key(kDeadKey, key_of(range.top), [&](uint32_t k) { return bin(value_of(k)) < border; }) - 1;
    if (lane == 0) w.to = to;
  } else if (wave == 2) {
    const uint32_t least = least_kept(Weigh(range.top, s.t, a.shift), range.top, s.m);
    if (lane == 0) w.least_kept = least;
  }
}

// Launch 4: the tokens that the border is among. top_k: all that reach its logit. top_p: those of its bin, and on
// a list of their own those ahead of it, as long as they are few.
template <int DT>
__global__ __launch_bounds__(256) void sample_collect_kernel(SampleArgs a) {
  __shared__ uint64_t list[2][kFew];
  __shared__ uint32_t have[2], base[2];
  const int r = blockIdx.x / a.splits, at = blockIdx.x % a.splits;
  const RowSettings s = settings(a, r);
  if (s.kind != kFront && s.kind != kShare) return;
  const RowReader<DT> row(a, r);
  RowWork& w = a.work[r];
  if (!(fabsf(row_range(a, w).top) < __builtin_inff())) return;
  constexpr int E = RowReader<DT>::E;
  const uint32_t from = w.from, to = w.to;
  const float low = value_of(from);
  const int g0 = at * a.per * a.chunk_units, g1 = min(row.units, (at + 1) * a.per * a.chunk_units);
  // lists of the workgroup: [0] the border's, [1] ahead of it, which is left alone once it is too long
  const float high = to == 0xFFFFFFFFu ? __builtin_inff() : value_of(to + 1);
  if (threadIdx.x < 2) have[threadIdx.x] = 0;
  __syncthreads();
  row.each(g0 + threadIdx.x, 256, g1, [&](int unit, const u32x4& u, int) {
    const float end = *(volatile uint32_t*)&have[1] > kFew ? high : __builtin_inff();
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float x = RowReader<DT>::raw(u, j);
      if (!(x >= low && x < end)) continue;
      const uint32_t k = key_of(x + 0.0f);
      const int which = k > to;
      const uint32_t n = atomicAdd(&have[which], 1u);
      const uint64_t p = place(k, unit * E - row.off + j);
      if (n < kFew) {
        list[which][n] = p;
      } else if (!which) {  // LDS is full: one by one
        const uint32_t at = atomicAdd(&w.n, 1u);
        if (at < kList) w.list[at] = p;
      }
    }
  });
  __syncthreads();
  // the row's lists: room for the workgroup's tokens, then they
  if (threadIdx.x < 2) {
    const uint32_t n = threadIdx.x ? have[1] : min(have[0], (uint32_t)kFew);
    base[threadIdx.x] = n ? atomicAdd(threadIdx.x ? &w.ahead : &w.n, n) : 0;
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x)
    for (uint32_t i = threadIdx.x; i < min(have[x], (uint32_t)kFew) && base[x] + i < (x ? kFew : kList); i += 256)
      w.list[x * kList + base[x] + i] = list[x][i];
}

// Launch 5, a workgroup a row: its token, or (top_p with many tokens kept) the last place kept.
template <int DT>
__global__ __launch_bounds__(1024) void sample_choose_kernel(SampleArgs a) {
  __shared__ SampleShared sm;
  const int r = blockIdx.x;
  const RowSettings s = settings(a, r);
  RowWork& w = a.work[r];
  int token = -1;
  if (s.kind == kGreedy) {
    const int lane = threadIdx.x & 63;
    const uint64_t best = wave_max64(lane < a.splits ? w.first[lane] : 0);
    if (best) token = token_of(best);
    if (threadIdx.x == 0) a.token[r] = token, w.done = 1;
    return;
  }
  const RowRange range = row_range(a, w);
  if (range.top != kDead) {
    const Weigh weigh(range.top, s.t, a.shift);
    const RowReader<DT> row(a, r);
    const bool list = s.kind == kFront || s.kind == kShare;
    const uint32_t n = list ? w.n : 0, ahead = s.kind == kShare ? w.ahead : 0;
    if (s.kind == kWhole || range.top == __builtin_inff() || n > kList) {
      if (threadIdx.x == 0) w.whole = 1;
      return;
    } else if (s.kind == kAll) {
      const float from = value_of(w.least_kept);
      const uint64_t mine = (int)threadIdx.x < a.chunks ? w.chunk[threadIdx.x] : 0;
      uint64_t all;
      if ((int)threadIdx.x < a.chunks) sm.chunk[threadIdx.x] = mine;
      scan_block<16>(mine, sm.red, &all);
      token = find<DT>(a, sm, row, pick_goal(s.u, all), [&](int, float x) { return weigh(x >= from ? x : kDead); });
    } else {
      const bool some = s.kind == kFront || n + ahead <= kFew;  // all that may be kept is at hand
      const int have = (int)(some ? n + ahead : n);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t i = threadIdx.x + 1024 * e;
        if ((int)i < have) sm.list[i] = i < n ? w.list[i] : w.list[kList + i - n];
      }
      __syncthreads();
      if (!some) {
        const int t = threadIdx.x;
        const Bins bin(value_of(min(w.to, key_of(range.top))), value_of(w.from), a.shift, __builtin_inf());
        uint64_t v[2], y[2];
        int at[2], border;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v[e] = t + 1024 * e < have ? sm.list[t + 1024 * e] : 0;
          const float x = value_of((uint32_t)(v[e] >> 32));
          at[e] = v[e] ? bin(x) : kBins;
          y[e] = v[e] ? weigh(x) : 0;
          sm.mass[t + 1024 * e] = 0;
        }
        __syncthreads();
        const uint64_t cut = last_by_mass(sm, weigh, v, y, at, w.before, w.goal, 0.0, &border);
        if (threadIdx.x == 0) w.cut = cut;
        return;
      }
      // what is on the lists is not all the row's weight, but the border's goal is of that
      const uint64_t goal = s.kind == kShare ? w.goal : 0;
      if (have <= 64 && threadIdx.x >= 64) return;
      if (have <= 64) token = choose_few(sm.list, weigh, have, s, goal);
      else token = choose(sm, weigh, Bins(range.top, value_of(w.from), a.shift, __builtin_inf()), have, s, goal, a.vocab);
    }
  }
  if (threadIdx.x == 0) a.token[r] = token, w.done = 1;
}

// What a token weighs that is at or before the cut of its row and enough for min_p.
struct Kept {
  Weigh weigh;
  float x, from;  // logit of the last token kept, and the least that min_p leaves
  int i;
  __device__ __forceinline__ Kept(const SampleArgs& a, const RowSettings& s, const RowWork& w, float top)
      : weigh(top, s.t, a.shift), x(value_of((uint32_t)(w.cut >> 32))), from(value_of(w.least_kept)), i(token_of(w.cut)) {}
  __device__ __forceinline__ uint64_t operator()(int at, float y) const {
    return weigh((y > x || (y == x && at <= i)) && y >= from ? y : kDead);
  }
};

// Launch 6: the kept tokens' weights, by chunks.
template <int DT>
__global__ __launch_bounds__(256) void sample_kept_kernel(SampleArgs a) {
  __shared__ u32x4 own[4 * 256];
  const int r = blockIdx.x / a.splits, at = blockIdx.x % a.splits;
  RowWork& w = a.work[r];
  if (w.done || w.whole) return;
  const RowSettings s = settings(a, r);
  const RowReader<DT> row(a, r);
  const Kept kept(a, s, w, row_range(a, w).top);
  const int c0 = at * a.per, c1 = min(a.chunks, c0 + a.per);
  for (int c = c0 + (threadIdx.x >> 6); c < c1; c += 4) {
    // equal logits are kept up to the cut's number: all of a chunk's, or none but in its own
    const int i0 = c * a.chunk_units * RowReader<DT>::E - row.off, i1 = i0 + a.chunk_units * RowReader<DT>::E;
    uint64_t v;
    if (kept.i >= i1 || kept.i < i0 || kept.from > kept.x) {
      const uint32_t k = key_of(kept.x) + (kept.i < i0 ? 1 : 0);
      const float from = fmaxf(value_of(k), kept.from);
      v = chunk_sum_from<DT>(a, row, c, kept.weigh, from, own + threadIdx.x);
    } else {
      v = chunk_sum<DT>(a, row, c, kept);
    }
    if ((threadIdx.x & 63) == 0) w.chunk[c] = v;
  }
}

// Last launch, a workgroup a row that has no token yet: rows whose kept weights are summed, and those with more
// tokens around the border than the list holds, with larger top_k or with an infinity, all of which is
// left to the workgroup. It is there for any row that needs it; with top_k most calls have none.
template <int DT>
__global__ __launch_bounds__(1024) void sample_last_kernel(SampleArgs a) {
  __shared__ SampleShared sm;
  const int r = blockIdx.x;
  RowWork& w = a.work[r];
  if (w.done) return;
  const RowSettings s = settings(a, r);
  const RowReader<DT> row(a, r);
  const RowRange range = row_range(a, w);
  int token;
  if (w.whole) {
    Sampler<DT> whole{a, sm, row, Weigh(range.top, s.t, a.shift), Bins(range.top, range.least, a.shift, s.t)};
    token = whole.whole(s);
  } else {
    const Kept kept(a, s, w, range.top);
    const uint64_t mine = (int)threadIdx.x < a.chunks ? w.chunk[threadIdx.x] : 0;
    uint64_t all;
    if ((int)threadIdx.x < a.chunks) sm.chunk[threadIdx.x] = mine;
    scan_block<16>(mine, sm.red, &all);
    token = find<DT>(a, sm, row, pick_goal(s.u, all), kept);
  }
  if (threadIdx.x == 0) a.token[r] = token;
}

constexpr int64_t kRowsAtOnce = 1024;  // rows of a batch of launches: 68 MB of workspace

// Workgroups of a row at most: enough for every CU, and several for the rows with more to do.
static int64_t most_splits(int64_t rows) { return std::min((int64_t)kSplits, std::max(2048 / rows, (int64_t)4)); }

template <int DT>
static int sample_rows(SampleArgs a, hipStream_t st) {
  const dim3 many((unsigned)(a.rows * a.splits)), one((unsigned)a.rows);
  // what no row can need is left out
  const bool greedy = !a.temperature && !(a.t > 0.0);
  const bool front = !greedy && (a.top_k || (a.k > 0 && a.k < a.vocab));
  const bool share = !greedy && (a.top_p || a.p < 1.0) && (a.top_k || !front);
  sample_range_kernel<DT><<<many, 256, 0, st>>>(a);
  if (!greedy) sample_weigh_kernel<DT><<<many, 256, 0, st>>>(a);
  if (share) sample_border_kernel<<<one, 256, 0, st>>>(a);
  if (front || share) sample_collect_kernel<DT><<<many, 256, 0, st>>>(a);
  sample_choose_kernel<DT><<<one, 1024, 0, st>>>(a);
  if (share) sample_kept_kernel<DT><<<many, 256, 0, st>>>(a);
  if (!greedy) sample_last_kernel<DT><<<one, 1024, 0, st>>>(a);
  CP_LAUNCHED("sampling");
  return CP_OK;
}

}  // namespace cp

extern "C" {

size_t cp_sample_ws_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1) return 0;
  const int64_t n = std::min(rows, cp::kRowsAtOnce);
  return (size_t)n * sizeof(cp::RowWork) + (size_t)n * cp::kMostPeaks * 4;
}

int cp_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_step, const void* u, int u_f64,
              const float* temperature, double temperature_all, const int32_t* top_k, int top_k_all, const float* top_p,
              double top_p_all, const float* min_p, double min_p_all, int32_t* token, void* ws, size_t ws_bytes,
              void* stream) {
  cp::clear_error();
  const int es = cp::dtype_bytes(dtype);
  if (!es) return cp::set_error(CP_ERR_ARG, "dtype code %d", dtype);
  if (vocab < 1 || vocab > 1 << 24) return cp::set_error(CP_ERR_SHAPE, "%lld tokens", (long long)vocab);
  if (rows < 0 || rows > 0x7FFFFFFF) return cp::set_error(CP_ERR_SHAPE, "%lld rows", (long long)rows);
  if (row_step < 0) return cp::set_error(CP_ERR_SHAPE, "negative stride of logits");
  if (rows == 0) return CP_OK;
  if (!logits || !u || !token) return cp::set_error(CP_ERR_ARG, "null logits / u / token");
  if (!cp::aligned(logits, es) || !cp::aligned(u, u_f64 ? 8 : 4))
    return cp::set_error(CP_ERR_ALIGN, "logits and u need their elements' alignment");
  if (!ws || ws_bytes < cp_sample_ws_bytes(rows, vocab))
    return cp::set_error(CP_ERR_WORKSPACE, "workspace of %zu bytes needs %zu", ws_bytes, cp_sample_ws_bytes(rows, vocab));
  if (!cp::aligned(ws, 256)) return cp::set_error(CP_ERR_ALIGN, "workspace needs 256-byte alignment");
  int bits = 0;
  while (((int64_t)1 << bits) < vocab) ++bits;
  const int per_unit = 16 / es;
  const int64_t units = (vocab + 2 * per_unit - 2) / per_unit;  // wherever a row begins in its first one
  int64_t chunk = cp::kChunkUnits;
  while ((units + chunk - 1) / chunk > cp::kChunks) chunk *= 2;
  for (int64_t r0 = 0; r0 < rows; r0 += cp::kRowsAtOnce) {
    cp::SampleArgs a;
    a.logits = (const char*)logits + r0 * row_step * es;
    a.step = row_step;
    a.rows = (int)std::min(rows - r0, cp::kRowsAtOnce);
    a.vocab = (int)vocab;
    a.shift = std::min(51, 62 - bits);
    a.u = (const char*)u + r0 * (u_f64 ? 8 : 4);
    a.u64 = u_f64;
    a.temperature = temperature ? temperature + r0 : nullptr;
    a.top_p = top_p ? top_p + r0 : nullptr;
    a.min_p = min_p ? min_p + r0 : nullptr;
    a.top_k = top_k ? top_k + r0 : nullptr;
    a.t = temperature_all;
    a.p = top_p_all;
    a.m = min_p_all;
    a.k = top_k_all;
    a.token = token + r0;
    a.work = (cp::RowWork*)ws;
    a.chunk_units = (int)chunk;
    a.chunks = (int)((units + chunk - 1) / chunk);
    const int64_t want = std::min((int64_t)a.chunks, cp::most_splits(a.rows));
    a.per = (int)((a.chunks + want - 1) / want);
    a.splits = (a.chunks + a.per - 1) / a.per;
    a.peaks = (uint32_t*)((char*)ws + a.rows * sizeof(cp::RowWork));
    a.peaks_each = 256 * cp::kPeaks;
    while (a.splits * a.peaks_each > cp::kMostPeaks) a.peaks_each /= 2;
    const int s = dtype == CP_F32    ? cp::sample_rows<CP_F32>(a, (hipStream_t)stream)
                  : dtype == CP_BF16 ? cp::sample_rows<CP_BF16>(a, (hipStream_t)stream)
                                     : cp::sample_rows<CP_F16>(a, (hipStream_t)stream);
    if (s) return s;
  }
  return CP_OK;
}

}  // extern "C"
