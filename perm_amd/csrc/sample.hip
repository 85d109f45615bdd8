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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lowbit.h"

namespace cp {

constexpr int kBins = 2048;    // of a histogram
constexpr int kList = 1024;    // tokens that are sorted at most: one a thread
constexpr int kChunks = 2048;  // pieces of a row whose weights are summed by themselves
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

// round(2^s e^((x - max) / T)) with scale = log2 e / T. 2^f for |f| <= 1/2 by its series to the 12th
// term, off by 6e-15; the product with 2^s rounds as 2^52 is added.
struct Weigh {
  double top, scale, unit;  // unit = 2^s
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const double r = fmax(((double)x - top) * scale, -64.0);
    const double n = rint(r), f = (r - n) * 0.69314718055994530942;
    double y = 1.0 / 39916800.0;
    y = __builtin_fma(y, f, 1.0 / 3628800.0);
    y = __builtin_fma(y, f, 1.0 / 362880.0);
    y = __builtin_fma(y, f, 1.0 / 40320.0);
    y = __builtin_fma(y, f, 1.0 / 5040.0);
    y = __builtin_fma(y, f, 1.0 / 720.0);
    y = __builtin_fma(y, f, 1.0 / 120.0);
    y = __builtin_fma(y, f, 1.0 / 24.0);
    y = __builtin_fma(y, f, 1.0 / 6.0);
    y = __builtin_fma(y, f, 0.5);
    y = __builtin_fma(y, f, 1.0);
    y = __builtin_fma(y, f, 1.0);
    const double two_n = __builtin_bit_cast(double, (uint64_t)((int64_t)(int)n + 1023) << 52);
    // x = max where that is an infinity: its difference is no number
    const double w = (double)x == top ? unit : y * (two_n * unit);
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) - 0x4330000000000000ull;
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
  // Element j of a unit: NaN as minus infinity, -0 as 0.
  static __device__ __forceinline__ float value(const u32x4& w, int j) {
    float x;
    if constexpr (DT == CP_F32) {
      const uint32_t b = w[j];
      x = __uint_as_float(b);
    } else {
      const uint32_t b = w[j >> 1];
      if constexpr (DT == CP_BF16)
        x = __uint_as_float(j & 1 ? b & 0xFFFF0000u : b << 16);
      else
        x = (float)__builtin_bit_cast(f16x2, b)[j & 1];
    }
    return fmaxf(x, kDead) + 0.0f;
  }
  // f(unit, its 16 bytes) for the units first, first + by, ...; four loads in flight.
  template <class F>
  __device__ __forceinline__ void each(int first, int by, F f) const {
    constexpr int U = 4;
    for (int g = first; g < units; g += U * by) {
      u32x4 w[U];
#pragma unroll
      for (int x = 0; x < U; ++x)
        if (g + x * by < units) w[x] = load(g + x * by);
#pragma unroll
      for (int x = 0; x < U; ++x)
        if (g + x * by < units) f(g + x * by, w[x]);
    }
  }
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int s) {
  const uint32_t lo = __shfl_xor((int)(uint32_t)v, s), hi = __shfl_xor((int)(v >> 32), s);
  return (uint64_t)hi << 32 | lo;
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

// Sum of v over the threads before this one, and over all 1024.
__device__ __forceinline__ uint64_t scan_block(uint64_t v, uint64_t* red, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t sum = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint64_t o = (uint64_t)(uint32_t)__shfl_up((int)(sum >> 32), s) << 32 | (uint32_t)__shfl_up((int)(uint32_t)sum, s);
    if (lane >= s) sum += o;
  }
  if (lane == 63) red[wave] = sum;
  __syncthreads();
  uint64_t base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    base += w < wave ? red[w] : 0;
    all += red[w];
  }
  __syncthreads();
  *total = all;
  return base + sum - v;
}

__device__ __forceinline__ uint64_t max_block(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint64_t o = shfl_xor64(v, s);
    v = o > v ? o : v;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) v = red[w] > v ? red[w] : v;
  __syncthreads();
  return v;
}

// The first n threads' values sorted, the largest first (threads past them: 0). Steps within a wave
// exchange by shuffles; n <= 64 needs no other.
__device__ __forceinline__ uint64_t sort_block(uint64_t v, int n, uint64_t* list) {
  const int t = threadIdx.x;
  int size = 64;
  while (size < n) size <<= 1;
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      uint64_t o;
      if (j < 64) {
        o = shfl_xor64(v, j);
      } else {
        list[t] = v;
        __syncthreads();
        o = list[t ^ j];
        __syncthreads();
      }
      const bool first = !(t & j), down = !(t & k);  // down: the larger one first
      v = (first == down) == (v > o) ? v : o;
    }
  return v;
}

// Threshold of a front: what is kept is every token whose place is at least this.
struct Cut {
  uint64_t place;
  bool list;  // LDS holds the n tokens at or before the cut's bin, unsorted
  int n;
};

template <int DT>
struct Sampler {
  const SampleArgs& a;
  SampleShared& sm;
  RowReader<DT> row;
  Weigh weigh;
  double unit;
  float top;      // largest logit
  float per_bin;  // bins a logit of one

  static constexpr int E = RowReader<DT>::E;

  // Bins of falling logits: monotone, as subtraction, product and conversion round monotonically. Where
  // the largest is an infinity, the others' differences or their products with 0 go to the last bin.
  __device__ __forceinline__ int bin(float x) const {
    return x == top ? 0 : min((int)fminf((top - x) * per_bin, 4e6f), kBins - 1);
  }

  template <class F>
  __device__ __forceinline__ void tokens(F f) const {
    row.each(threadIdx.x, 1024, [&](int unit, const u32x4& w) {
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
    const uint64_t c = scan_block(c0 + c1, sm.red, &all), m = scan_block(m0 + m1, sm.red, &all);
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
  __device__ __forceinline__ uint32_t least_key(int b) const {
    uint32_t lo = key_of(kDead) + 1, hi = key_of(top);  // bin(hi) = 0 <= b
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (bin(value_of(mid)) <= b) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }

  // Of the tokens at or above `cut`, the place of the last one kept: by_count tokens, or those before which
  // less than by_mass lies. Afterwards *kept is their weight (by_mass only).
  //
  // A histogram finds the bin the border lies in; the bin's keys are split again until its tokens fit
  // the list, or are all equal.
  __device__ __forceinline__ Cut front(uint64_t cut, uint64_t by_count, uint64_t by_mass, int at, uint64_t count,
                                       uint64_t mass) {
    uint32_t hi = at == 0 ? key_of(top) : least_key(at - 1) - 1, lo = least_key(at);
    for (;;) {
      int n;
      const uint64_t in_bin = sm.count[at];
      if (count + in_bin <= kList) {  // everything down to the border fits
        collect(lo, 0xFFFFFFFFu, cut, &n);
        return {0, true, n};
      }
      if (in_bin <= kList) {
        collect(lo, hi, cut, &n);
        const uint64_t v = sort_block(threadIdx.x < n ? sm.list[threadIdx.x] : 0, n, sm.list);
        const uint64_t w = threadIdx.x < n ? weigh(value_of((uint32_t)(v >> 32))) : 0;
        uint64_t all;
        const uint64_t before = mass + scan_block(w, sm.red, &all);
        const bool keep = threadIdx.x < n && (by_count ? count + threadIdx.x < by_count : before < by_mass);
        // the last kept: the smallest place
        const uint64_t last = ~max_block(keep ? ~v : 0, sm.red);
        return {last, false, 0};
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
          if (by_mass) atomicAdd((unsigned long long*)&sm.mass[b], (unsigned long long)weigh(x));
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
      const uint64_t w = weigh(value_of(hi));
      need = w ? (by_mass - mass + w - 1) / w : 1;
    }
    return {nth(hi, cut, need), false, 0};
  }

  // Elements of a chunk, a power of two of the units a wave takes in a step.
  __device__ __forceinline__ int chunk_shift() const {
    int s = 6;
    while (((row.units - 1) >> s) >= kChunks) ++s;
    return s;
  }

  // Sums value(i, x) over chunks of the row into sm.chunk, then finds the chunk in which the sum in the
  // order of numbers passes `goal`: the number of the first token at which it does.
  template <class F>
  __device__ __forceinline__ void chunk_sums(F value) {
    for (int i = threadIdx.x; i < kChunks; i += 1024) sm.chunk[i] = 0;
    __syncthreads();
    const int s = chunk_shift();
    for (int unit = threadIdx.x; unit - (int)(threadIdx.x & 63) < row.units; unit += 1024) {  // whole waves
      const int i0 = unit * E - row.off;
      uint64_t v = 0;
      if (unit < row.units) {
        const u32x4 w = row.load(unit);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float x = RowReader<DT>::value(w, j);
          if (x != kDead) v += value(i0 + j, x);
        }
      }
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) v += shfl_xor64(v, k);
      if ((threadIdx.x & 63) == 0) atomicAdd((unsigned long long*)&sm.chunk[unit >> s], (unsigned long long)v);
    }
    __syncthreads();
  }

  template <class F>
  __device__ __forceinline__ int find(uint64_t goal, F value) {
    const int i = 2 * threadIdx.x;
    uint64_t all;
    const uint64_t c0 = sm.chunk[i], c1 = sm.chunk[i + 1], c = scan_block(c0 + c1, sm.red, &all);
    if (c <= goal && c + c0 > goal) sm.pick[0] = i, sm.pick[1] = c;
    else if (c + c0 <= goal && c + c0 + c1 > goal) sm.pick[0] = i + 1, sm.pick[1] = c + c0;
    __syncthreads();
    const int at = (int)sm.pick[0], s = chunk_shift();
    if (threadIdx.x < 64) {  // 64 units a step, in order
      uint64_t base = sm.pick[1];
      const int end = min(row.units, (at + 1) << s);
      for (int g = (at << s) + threadIdx.x; __any(g < end); g += 64) {
        uint64_t v[E], sum = 0;
        u32x4 w = {};
        if (g < end) w = row.load(g);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float x = RowReader<DT>::value(w, j);
          v[j] = g < end && x != kDead ? value(g * E - row.off + j, x) : 0;
          sum += v[j];
        }
        uint64_t incl = sum;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
          const uint64_t o =
              (uint64_t)(uint32_t)__shfl_up((int)(incl >> 32), k) << 32 | (uint32_t)__shfl_up((int)(uint32_t)incl, k);
          if ((int)threadIdx.x >= k) incl += o;
        }
        const unsigned long long hit = __ballot(base + incl > goal);
        if (hit) {
          const int l = __ffsll(hit) - 1;
          if ((int)threadIdx.x == l) {
            uint64_t b = base + incl - sum;
            int j = 0;
#pragma unroll
            for (int x = 0; x < E; ++x) {
              b += v[x];
              if (b <= goal) j = x + 1;
            }
            sm.pick[2] = (uint64_t)(g * E - row.off + min(j, E - 1));
          }
          break;
        }
        base += (uint64_t)(uint32_t)__shfl((int)(incl >> 32), 63) << 32 | (uint32_t)__shfl((int)(uint32_t)incl, 63);
      }
    }
    __syncthreads();
    return (int)sm.pick[2];
  }

  // The place of the need'th token with this key at or above `cut`, by number.
  __device__ __forceinline__ uint64_t nth(uint32_t key, uint64_t cut, uint64_t need) {
    auto one = [&](int i, float x) -> uint64_t { return key_of(x) == key && place(key, i) >= cut; };
    chunk_sums(one);
    uint64_t v = 0, all;
    for (int i = threadIdx.x; i < kChunks; i += 1024) v += sm.chunk[i];
    scan_block(v, sm.red, &all);
    if (all == 0) return cut;  // no such token: not reached
    return place(key, find(min(need, all) - 1, one));
  }

  // The tokens of the list, sorted, are all that is left to choose from.
  __device__ __forceinline__ int choose(int n, uint64_t k, double p, double m, double u) {
    const int t = threadIdx.x;
    const uint64_t v = sort_block(t < n ? sm.list[t] : 0, n, sm.list);
    uint64_t total, kept;
    const bool in = t < n && (k == 0 || (uint64_t)t < k);
    const uint64_t w = in ? weigh(value_of((uint32_t)(v >> 32))) : 0;
    const uint64_t before = scan_block(w, sm.red, &total);
    const bool keep = in && (t == 0 || ((!(p < 1.0) || before < mass_goal(p, total)) && (double)w >= m * unit));
    scan_block(keep ? w : 0, sm.red, &kept);
    const uint64_t goal = pick_goal(u, kept);
    __syncthreads();
    sm.mass[t] = keep ? w : 0;
    // by rising number, the kept ones first
    const uint64_t by_number = sort_block(keep ? (uint64_t)(uint32_t)v << 32 | (uint32_t)t : 0, n, sm.list);
    const uint64_t mine = by_number ? sm.mass[(uint32_t)by_number] : 0;
    const uint64_t b = scan_block(mine, sm.red, &total);
    if (b <= goal && b + mine > goal) sm.pick[2] = (uint64_t)(0xFFFFFFFFu - (uint32_t)(by_number >> 32));
    __syncthreads();
    return (int)sm.pick[2];
  }

  // Least whole number that is no less than p times the sum, and at least 1: the first token stays.
  static __device__ __forceinline__ uint64_t mass_goal(double p, uint64_t total) {
    const double g = ceil(fmax(p, 0.0) * (double)total);
    return g >= (double)total ? total : max((uint64_t)g, (uint64_t)1);
  }
  static __device__ __forceinline__ uint64_t pick_goal(double u, uint64_t total) {
    const double g = floor(fmax(u, 0.0) * (double)total);
    return g >= (double)(total - 1) ? total - 1 : (uint64_t)g;
  }
};

// A workgroup a row.
template <int DT>
__global__ __launch_bounds__(1024) void sample_kernel(SampleArgs a) {
  __shared__ SampleShared sm;
  const int r = blockIdx.x;
  const double t = a.temperature ? (double)a.temperature[r] : a.t;
  const double p = a.top_p ? (double)a.top_p[r] : a.p, m0 = a.min_p ? (double)a.min_p[r] : a.m;
  const double m = m0 > 0.0 ? fmin(m0, 1.0) : 0.0;
  const double u = a.u64 ? ((const double*)a.u)[r] : (double)((const float*)a.u)[r];
  uint64_t k = max(a.top_k ? a.top_k[r] : a.k, 0);
  if (k >= (uint64_t)a.vocab) k = 0;
  Sampler<DT> s{a, sm, RowReader<DT>(a, r)};
  if (!(t > 0.0)) {
    uint64_t best = 0;
    s.tokens([&](int i, float x) {
      const uint64_t v = place(key_of(x), i);
      best = v > best ? v : best;
    });
    best = max_block(best, sm.red);
    if (threadIdx.x == 0) a.token[r] = best ? token_of(best) : -1;
    return;
  }
  float top = kDead, least = __builtin_inff();
  uint32_t alive = 0;
  s.tokens([&](int, float x) {
    top = fmaxf(top, x), least = fminf(least, x);
    ++alive;
  });
  top = value_of((uint32_t)max_block(key_of(top), sm.red));
  least = value_of(~(uint32_t)max_block(~key_of(least), sm.red));
  uint64_t all;
  scan_block(alive, sm.red, &all);
  if (all == 0) {
    if (threadIdx.x == 0) a.token[r] = -1;
    return;
  }
  if (k >= all) k = 0;
  s.unit = __builtin_bit_cast(double, (uint64_t)(a.shift + 1023) << 52);
  s.weigh = {(double)top, 1.4426950408889634074 / t, s.unit};
  s.top = top;
  // bins down to the least logit, or to where weights are 0
  const double span = fmin((double)top - (double)least, (double)(a.shift + 2) * 0.6931471805599453 * t);
  s.per_bin = span > 0.0 ? (float)fmin((double)kBins / span, 3e38) : 0.0f;
  if (!(s.per_bin > 0.0f)) s.per_bin = 0.0f;
  uint64_t cut = 0;
  if (k) {
    s.clear_bins();
    s.tokens([&](int, float x) { atomicAdd(&sm.count[s.bin(x)], 1u); });
    __syncthreads();
    int at;
    uint64_t count, mass;
    s.border(k, 0, &at, &count, &mass);
    const Cut c = s.front(0, k, 0, at, count, 0);
    if (c.list) {
      const int token = s.choose(c.n, k, p, m, u);
      if (threadIdx.x == 0) a.token[r] = token;
      return;
    }
    cut = c.place;
  }
  if (p < 1.0) {
    s.clear_bins();
    s.tokens([&](int i, float x) {
      if (place(key_of(x), i) < cut) return;
      const int b = s.bin(x);
      atomicAdd(&sm.count[b], 1u);
      atomicAdd((unsigned long long*)&sm.mass[b], (unsigned long long)s.weigh(x));
    });
    __syncthreads();
    uint64_t v = 0, total;
    for (int i = threadIdx.x; i < kBins; i += 1024) v += sm.mass[i];
    scan_block(v, sm.red, &total);
    const uint64_t goal = Sampler<DT>::mass_goal(p, total);
    int at;
    uint64_t count, mass;
    s.border(0, goal, &at, &count, &mass);
    const Cut c = s.front(cut, 0, goal, at, count, mass);
    if (c.list) {
      // the list holds tokens past the border, too: whole bins. Their sum is not the row's
      const int t0 = threadIdx.x;
      const uint64_t place = sort_block(t0 < c.n ? sm.list[t0] : 0, c.n, sm.list);
      const uint64_t w = t0 < c.n ? s.weigh(value_of((uint32_t)(place >> 32))) : 0;
      uint64_t sum;
      const uint64_t before = scan_block(w, sm.red, &sum);
      const bool keep = t0 < c.n && (t0 == 0 || before < goal);
      uint64_t n;
      scan_block(keep, sm.red, &n);
      __syncthreads();
      sm.list[t0] = keep ? place : 0;
      __syncthreads();
      const int token = s.choose((int)n, 0, 1.0, m, u);
      if (threadIdx.x == 0) a.token[r] = token;
      return;
    }
    cut = c.place;
  }
  const double least_w = m * s.unit;
  auto value = [&](int i, float x) -> uint64_t {
    if (place(key_of(x), i) < cut) return 0;
    const uint64_t w = s.weigh(x);
    return (double)w >= least_w || x == top ? w : 0;
  };
  s.chunk_sums(value);
  uint64_t v = 0, total;
  for (int i = threadIdx.x; i < kChunks; i += 1024) v += sm.chunk[i];
  scan_block(v, sm.red, &total);
  const int token = s.find(Sampler<DT>::pick_goal(u, total), value);
  if (threadIdx.x == 0) a.token[r] = token;
}

}  // namespace cp

extern "C" {

int cp_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_step, const void* u, int u_f64,
              const float* temperature, double temperature_all, const int32_t* top_k, int top_k_all, const float* top_p,
              double top_p_all, const float* min_p, double min_p_all, int32_t* token, void* stream) {
  cp::clear_error();
  const int es = cp::dtype_bytes(dtype);
  if (!es) return cp::set_error(CP_ERR_ARG, "dtype code %d", dtype);
  if (vocab < 1 || vocab > 1 << 24) return cp::set_error(CP_ERR_SHAPE, "%lld tokens", (long long)vocab);
  if (rows < 0 || rows > cp::most_workgroups(1024)) return cp::set_error(CP_ERR_SHAPE, "%lld rows", (long long)rows);
  if (row_step < 0) return cp::set_error(CP_ERR_SHAPE, "negative stride of logits");
  if (rows == 0) return CP_OK;
  if (!logits || !u || !token) return cp::set_error(CP_ERR_ARG, "null logits / u / token");
  if (!cp::aligned(logits, es) || !cp::aligned(u, u_f64 ? 8 : 4))
    return cp::set_error(CP_ERR_ALIGN, "logits and u need their elements' alignment");
  cp::SampleArgs a;
  a.logits = logits;
  a.step = row_step;
  a.rows = (int)rows;
  a.vocab = (int)vocab;
  int bits = 0;
  while (((int64_t)1 << bits) < vocab) ++bits;
  a.shift = std::min(51, 62 - bits);
  a.u = u;
  a.u64 = u_f64;
  a.temperature = temperature;
  a.top_p = top_p;
  a.min_p = min_p;
  a.top_k = top_k;
  a.t = temperature_all;
  a.p = top_p_all;
  a.m = min_p_all;
  a.k = top_k_all;
  a.token = token;
  const dim3 grid((unsigned)rows);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CP_F32) cp::sample_kernel<CP_F32><<<grid, 1024, 0, st>>>(a);
  if (dtype == CP_BF16) cp::sample_kernel<CP_BF16><<<grid, 1024, 0, st>>>(a);
  if (dtype == CP_F16) cp::sample_kernel<CP_F16><<<grid, 1024, 0, st>>>(a);
  CP_LAUNCHED("sampling");
  return CP_OK;
}

}  // extern "C"
