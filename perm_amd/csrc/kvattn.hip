// Attention over the paged 8-bit cache on gfx950.
//
// Row i of a sequence with n query rows and len tokens sits at position p = len - n + i and
// sees token j where j < len, j <= p (causal) and j > p - window (window > 0). With K and V
// codes in e4m3 and power-of-two scales ks, vs of each page and head, in base 2:
//
//     t_j = (q . kcode_j) * ks_j * scale * log2 e + log2 vs_j
//     w_j = 2^(t_j - m + 11),  m the running maximum of t within four binades
//     out = sum_j w_j vcode_j / sum_j (w_j / vs_j)
//
// V's scale rides in the exponent, so the codes feed the matrix cores unscaled and w is at
// most 2^15 whatever the scales are. Scores, m, the sum and the output accumulate in float32. K
// codes become q's own 16-bit type, which holds e4m3 exactly.
//
// w is rounded as the second product's operand, and must not be lost for being small beside
// others: where a first token takes most of the softmax and has no values, or a page with a large
// V scale holds zeros in a column, small weights are all that the result consists of. It is either
// one float16, which has 11 bits of a weight down to 2^-14, 25 binades below the running
// maximum; or two bfloat16 terms, 16 bits of it down to 2^-126, for twice the MFMAs. Few query rows
// always take the two terms (bound by reading the cache, they cost nothing); of many rows, a wave
// takes them from the first unit on in which one of its rows sees a smaller weight.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kvcache.h"
#include "lowbit.h"

namespace cp {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;       // tokens per step of a wave
constexpr float kNegInf = -__builtin_inff();
// Weights are 2^kLift above 2^(t - m), which uses float16's range up to 2^15: m moves when a t
// passes it by kLag. A t more than kDeep below m has a weight below float16's normal range.
constexpr float kLift = 11.0f, kLag = 4.0f, kDeep = kLift + 14.0f;

struct AttnArgs {
  KvCacheArgs c;
  const void* q;                // [rows][q heads][d]
  int64_t q_row, q_head;
  const int* lens;              // [batch]
  void* out;                    // [rows][q heads][d]
  float* lse;                   // [rows][q heads] or null
  // splits > 1, a row being one of a sequence's and head: [row][splits][d] sums, then
  // [row][splits] pairs (m, l), then [row] int: how many splits the row used, 0 if it is done
  float* part;
  int64_t rows;
  int group;                    // q heads per kv head
  int causal, window, splits;
  int least;                    // tiles of a split at least
  float scale;                  // softmax scale * log2 e
};

struct SplitParts {
  float *sums, *ml;
  int* used;
};

__host__ __device__ inline SplitParts split_parts(const AttnArgs& a) {
  const int64_t n = a.rows * a.group * a.c.heads * a.splits;
  float* ml = a.part + n * a.c.d;
  return {a.part, ml, reinterpret_cast<int*>(ml + 2 * n)};
}

// Results of the rows [0, lead) and [tail, end): 0, lse -inf, nothing to join. Workgroup `at` of `of`.
template <int DT>
__device__ __forceinline__ void attn_clear(const AttnArgs& a, int64_t lead, int64_t tail, int64_t end, int at, int of) {
  const int64_t per = (int64_t)a.group * a.c.heads, skip = (tail - lead) * per;
  for (int64_t i = (int64_t)at * blockDim.x + threadIdx.x; i < end * per - skip; i += (int64_t)of * blockDim.x) {
    const int64_t r = i < lead * per ? i : i + skip;
    typename Elem<DT>::T* p = (typename Elem<DT>::T*)a.out + r * a.c.d;
    for (int x = 0; x < a.c.d; x += 8) *reinterpret_cast<u32x4*>(p + x) = u32x4{0, 0, 0, 0};
    if (a.lse) a.lse[r] = kNegInf;
    if (a.splits > 1) split_parts(a).used[r] = 0;
  }
}

// What a workgroup without rows of its own does. at: its item past the end, or -1 for a sequence
// whose rows are not all among the call's: those that are have no results either.
template <int DT>
__device__ __forceinline__ void attn_unowned(const AttnArgs& a, const KvBatch& bt, int at, int of, int piece, int64_t row0,
                                             int n_b) {
  const int pieces = a.c.heads * a.splits;
  if (at >= 0) {
    if (!bt.offsets) return;
    const KvUnowned u = kv_unowned(bt, a.rows);
    attn_clear<DT>(a, u.lead, u.tail, a.rows, at * pieces + piece, of * pieces);
  } else {
    const int64_t end = min(row0 + n_b, a.rows), from = min(max(row0, (int64_t)0), end);
    attn_clear<DT>(a, 0, from, end, piece, pieces);
  }
}

// Eight e4m3 codes in q's type / in float16 (both exact).
template <int DT>
__device__ __forceinline__ u32x4 codes_to_16(uint32_t a, uint32_t b) {
  u32x4 r;
  if constexpr (DT == CP_BF16) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
  }
  return r;
}

template <int DT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == CP_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// Two weights as bfloat16 terms: hi rounded, lo the rest rounded.
struct Weights2 {
  uint32_t hi, lo;
};
__device__ __forceinline__ Weights2 weights2(float e0, float e1) {
  const uint32_t hi = pack2<CP_BF16>(e0, e1);
  return {hi, pack2<CP_BF16>(e0 - __uint_as_float(hi << 16), e1 - __uint_as_float(hi & 0xFFFF0000u))};
}

// What sums over an old maximum m are multiplied by when it moves to mn: the square of this. The
// sum of weights takes it in two steps, being as large as V's scales are small (up to 2^60 times
// the weights), and outlives a move of more than 126 binades.
__device__ __forceinline__ float half_move(float m, float mn) {
  return exp2_fast(0.5f * (m - (mn == kNegInf ? 0.0f : mn)));
}

// Log-sum-exp of a row whose weights, lifted by 2^kLift, sum to l over the maximum m.
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? kNegInf : (m - kLift + __builtin_amdgcn_logf(l)) / kLog2e;
}

// Bytes of w that are NaN codes (0x7F or 0xFF) as 0x80 flags: 0x7F is the only magnitude
// that carries out of seven bits when one is added.
__device__ __forceinline__ uint32_t nan_flags(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// Few query rows: a workgroup takes up to 16 (row, head of the group) pairs of one kv head
// and one range of tokens; its four waves walk the range 32 tokens at a time in turn and
// join at the end. Bound by reading the cache, and for short ranges by the latencies a
// workgroup starts with (length, page numbers, codes), which four workgroups on a CU hide
// better than longer strides in fewer of them: hence small tiles and at most 128 registers.
// One token of 32 heads on 131072 tokens: 268 MB in 49 us, 5.4 TB/s. 64 sequences of up to 4096
// tokens: 174 MB in 41 us, 34 with equal lengths; the longest sequence's splits end last. Weights in
// two terms cost 1 % at 128 columns, 8 % at 80, whose products are 128 wide all the same.
//
// K is the A operand (16 tokens x 32 columns), q the B operand, so a lane's scores belong to
// one query row (lane % 16), and its group lane / 16 owns 8 consecutive tokens of the tile:
// score (t, i) of the lane is token 8 (lane / 16) + 4 t + i. Those are the eight-token runs
// the second product's operands hold, so the weights go from one product to the other
// without leaving their lanes.
constexpr int kFewTile = 32;

template <int DT, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 2 : 4) void attn_few_kernel(AttnArgs a, KvBatch bt, int items) {
  constexpr int NC = DP / 64, ND = DP / 16;
  __shared__ float sm_m[4][16], sm_l[4][16];
  __shared__ __align__(16) float sm_o[4][16][DP + 4];
  const KvCacheArgs& c = a.c;
  const int split = (int)(blockIdx.x % a.splits);
  const int h = (int)(blockIdx.x / a.splits % c.heads);
  int b, item, n_b;
  int64_t row0;
  const int at = (int)(blockIdx.x / a.splits / c.heads), piece = h * a.splits + split;
  if (!kv_locate(bt, at, [&](int, int n) { return (int)(((int64_t)n * a.group + 15) / 16); }, &b, &item, &row0, &n_b))
    return attn_unowned<DT>(a, bt, item, items - at + item, piece, 0, 0);
  if (row0 < 0 || row0 + n_b > a.rows) {
    if (item == 0) attn_unowned<DT>(a, bt, -1, 0, piece, row0, n_b);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int d = c.d, blk = c.block, lb = 31 - __clz(c.block);  // block is a power of two
  // rows sit at the end of len tokens, of which the table holds the first
  const int len = max(a.lens[b], 0), held = (int)min((int64_t)len, (int64_t)c.max_pages * blk);

  // this lane's query row
  const int64_t r = (int64_t)item * 16 + col;
  const bool real = r < (int64_t)n_b * a.group;
  const int qi = (int)(r / a.group), qh = h * a.group + (int)(r % a.group);
  const int64_t pos = (int64_t)len - n_b + qi;
  int hi = real ? (a.causal ? (int)max((int64_t)0, min((int64_t)held, pos + 1)) : held) : 0;
  int lo = a.window > 0 ? (int)max((int64_t)0, pos - a.window + 1) : 0;
  if (lo >= hi) lo = hi = 0;
  // tokens any row of the workgroup sees
  int jhi = hi, jlo = hi > lo ? lo : 0x7FFFFFFF;
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) {
    jhi = max(jhi, __shfl_xor(jhi, s));
    jlo = min(jlo, __shfl_xor(jlo, s));
  }
  jhi = __builtin_amdgcn_readfirstlane(jhi);
  jlo = min(__builtin_amdgcn_readfirstlane(jlo), jhi);
  const int t0 = jlo / kFewTile, nt = (jhi + kFewTile - 1) / kFewTile - t0;
  // a row's tiles are shared evenly by the splits; one of few tiles uses few of them
  const int per = max((nt + a.splits - 1) / a.splits, a.least), used = (nt + per - 1) / per;
  if (split > 0 && split >= used) return;
  const int tb = t0 + split * per, te = min(t0 + nt, tb + per);

  u32x4 qf[NC][2];
  {
    typedef typename Elem<DT>::T T;
    const T* qp = (const T*)a.q + (real ? (row0 + qi) * a.q_row + (int64_t)qh * a.q_head : 0);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const bool in = real && 64 * k + 16 * g < d;
      const u32x4 z = {0, 0, 0, 0};
      const T* p = qp + (64 * k + 16 * g < d ? 64 * k + 16 * g : 0);
      qf[k][0] = *reinterpret_cast<const u32x4*>(p);
      qf[k][1] = *reinterpret_cast<const u32x4*>(p + 8);
      if (!in) qf[k][0] = qf[k][1] = z;
    }
  }
  f32x4 o[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) o[i] = f32x4{0, 0, 0, 0};
  float m = kNegInf, l = 0.0f;
  const int* tab = c.table + (int64_t)b * c.max_pages;
  // columns past d read the row's first ones instead: their q is 0, and a NaN there makes the
  // score NaN anyway
  int kcol[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) kcol[k] = 64 * k + 16 * g < d ? 64 * k + 16 * g : 0;
  uint64_t marked = 0;  // bit 4 i + k: result (i, k) of this lane has seen a NaN code
  u32x2* const mine = reinterpret_cast<u32x2*>(&sm_o[wave][0][0]) + lane;

  // pages of the token runs this lane reads: K rows by lane % 16 / 4, V and the scores' scales
  // by lane / 16. Looked up a tile ahead.
  const int lastj = max(jhi - 1, 0);
  auto page = [&](int j) { return tab[min(j, lastj) >> lb]; };
  int pk = 0, pv = 0;
  if (tb + wave < te) {
    pk = page((tb + wave) * kFewTile + 8 * (col >> 2));
    pv = page((tb + wave) * kFewTile + 8 * g);
  }
#pragma clang loop unroll(disable)
  for (int tile = tb + wave; tile < te; tile += 4) {
    const int jk = tile * kFewTile + 8 * (col >> 2), jv = tile * kFewTile + 8 * g;
    const bool hk = (unsigned)pk < (unsigned)c.pages, have = (unsigned)pv < (unsigned)c.pages;
    const int64_t hv = (int64_t)(have ? pv : 0) * c.heads + h;
    const uint8_t* kp = c.k + ((int64_t)(hk ? pk : 0) * c.heads + h) * blk * d + ((jk & (blk - 1)) + (col & 3)) * d;
    const uint8_t* vp = c.v + hv * blk * d + col * blk + (jv & (blk - 1));
    u32x4 kk[2][NC];
    u32x2 vv[ND];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < NC; ++k) kk[t][k] = *reinterpret_cast<const u32x4*>(kp + 4 * t * d + kcol[k]);
    const float ks0 = c.k_scale[hv], vs0 = c.v_scale[hv];
#pragma unroll
    for (int i = 0; i < ND; ++i) {  // rows past d repeat the last one and are dropped
      vv[i] = *reinterpret_cast<const u32x2*>(vp);
      if (16 * (i + 1) < d) vp += 16 * blk;
    }
    pk = page(jk + 4 * kFewTile);
    pv = page(jv + 4 * kFewTile);
    // no page: page 0's codes, which no row sees, but its scales may be anything and would reach them
    const float ks = have ? ks0 : 1.0f, vs = have ? vs0 : 1.0f;
    f32x4 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        sc[t] = mfma16<DT>(codes_to_16<DT>(kk[t][k][0], kk[t][k][1]), qf[k][0], sc[t]);
        sc[t] = mfma16<DT>(codes_to_16<DT>(kk[t][k][2], kk[t][k][3]), qf[k][1], sc[t]);
      }
    }
    const float kc = ks * a.scale;
    const float lv = (float)((int)(__float_as_uint(vs) >> 23) - 127);
    bool edge = false;  // a token of this lane that its row does not see
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = jv + 4 * t + i;
        const bool see = have && j >= lo && j < hi;
        edge |= !see;
        sc[t][i] = see ? sc[t][i] : kNegInf;
      }
    // kc > 0: the largest t of the lane's run comes from its largest raw score
    float tm = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                     fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    tm = __builtin_fmaf(tm, kc, lv);
    // the running maximum moves only when a t passes it by kLag, so the row's lanes seldom have
    // to exchange their largest and rescale the outputs
    if (__any(tm > m + kLag)) {
      tm = fmaxf(tm, __shfl_xor(tm, 16));
      tm = fmaxf(tm, __shfl_xor(tm, 32));
      const float mn = fmaxf(m, tm), ah = half_move(m, mn), al = ah * ah;
      m = mn;
      l = l * ah * ah;
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] *= al;
    }
    // w / vs, the sum's term, and w from it: where V's scales are far apart w may fall out of
    // float32's range beside the other results, but its term does not beside the sum
    const float off = kLift - (m == kNegInf ? 0.0f : m);
    u32x4 wh, wl;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const float e0 = exp2_fast(__builtin_fmaf(sc[t][i], kc, off));
        const float e1 = exp2_fast(__builtin_fmaf(sc[t][i + 1], kc, off));
        sum += e0 + e1;
        const Weights2 x = weights2(e0 * vs, e1 * vs);
        wh[2 * t + (i >> 1)] = x.hi, wl[2 * t + (i >> 1)] = x.lo;
      }
    l += sum;
    // a code that a row does not see must not reach it, not even as 0 * NaN: NaN codes are
    // taken out of the product and put back into the rows that do see them
    bool nan = false;
    if (__any(edge)) {
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < ND; ++i) any |= nan_flags(vv[i][0]) | nan_flags(vv[i][1]);
      nan = __any(any != 0);
      if (nan) {
        // through the wave's LDS in a loop: unrolled in registers, this rare path would make
        // the common one spill
#pragma unroll
        for (int i = 0; i < ND; ++i) mine[64 * i] = vv[i];
        u32x4 one = {0, 0, 0, 0};  // 1.0 where this lane's row sees the token
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = jv + e;
          if (have && j >= lo && j < hi) one[e >> 1] |= 0x3C00u << (16 * (e & 1));
        }
#pragma clang loop unroll(disable)
        for (int i = 0; i < ND; ++i) {
          u32x2 y = mine[64 * i];
          const uint32_t f0 = nan_flags(y[0]) >> 7, f1 = nan_flags(y[1]) >> 7;
          y[0] &= ~(f0 * 0xFFu);
          y[1] &= ~(f1 * 0xFFu);
          mine[64 * i] = y;
          // e4m3 1.0 where the code was NaN
          const f32x4 cnt = mfma16<CP_F16>(codes_to_16<CP_F16>(f0 * 0x38u, f1 * 0x38u), one, f32x4{0, 0, 0, 0});
#pragma unroll
          for (int k = 0; k < 4; ++k) marked |= cnt[k] > 0.0f ? (uint64_t)1 << (4 * i + k) : 0;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      u32x2 y = vv[i];
      if (nan) y = mine[64 * i];
      const u32x4 x = codes_to_16<CP_BF16>(y[0], y[1]);
      o[i] = mfma16<CP_BF16>(x, wh, o[i]);
      o[i] = mfma16<CP_BF16>(x, wl, o[i]);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) sm_m[wave][col] = m, sm_l[wave][col] = l;
  if (__any(marked != 0)) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = marked >> (4 * i + k) & 1 ? __builtin_nanf("") : o[i][k];
  }
#pragma unroll
  for (int i = 0; i < ND; ++i) *reinterpret_cast<f32x4*>(&sm_o[wave][col][16 * i + 4 * g]) = o[i];
  __syncthreads();
  // join the four waves: thread -> row threadIdx / 16, four columns at a time
  const int row = threadIdx.x >> 4, c0 = threadIdx.x & 15;
  const int64_t rr = (int64_t)item * 16 + row;
  if (rr >= (int64_t)n_b * a.group) return;
  float mm = kNegInf, f[4], ll = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm_m[w][row]);
  const float ms = mm == kNegInf ? 0.0f : mm;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float fh = half_move(sm_m[w][row], ms);
    f[w] = fh * fh;
    ll += sm_l[w][row] * fh * fh;
  }
  const int64_t orow = (row0 + rr / a.group) * ((int64_t)a.group * c.heads) + h * a.group + rr % a.group;
  const SplitParts sp = split_parts(a);
  if (a.splits > 1 && split == 0 && c0 == 0) sp.used[orow] = used > 1 ? used : 0;
  float* p = sp.sums + (orow * a.splits + split) * d;
  typename Elem<DT>::T* op = (typename Elem<DT>::T*)a.out + orow * d;
  const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;  // a row that saw nothing: 0
  for (int x = 4 * c0; x < d; x += 64) {
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(&sm_o[w][row][x]) * f[w];
    if (used > 1) {
      *reinterpret_cast<f32x4*>(p + x) = v;
    } else {
      u32x2 y;
      y[0] = pack2<DT>(v[0] * inv, v[1] * inv);
      y[1] = pack2<DT>(v[2] * inv, v[3] * inv);
      *reinterpret_cast<u32x2*>(op + x) = y;
    }
  }
  if (c0 != 0) return;
  if (used > 1) {
    float* pm = sp.ml + (orow * a.splits + split) * 2;
    pm[0] = mm, pm[1] = ll;
  } else if (a.lse) {
    a.lse[orow] = row_lse(mm, ll);
  }
}

// Many query rows: a workgroup takes 128 (row, head of the group) pairs of one kv head, 32 a
// wave, and walks its range of tokens 64 at a time. The tile's K and V codes are staged in
// LDS a tile ahead by loads that write LDS directly, and every wave turns the codes it reads
// into 16 bits itself. The products are v_mfma_f32_32x32x16 with K and V as the A operand, so
// a lane's scores belong to one query row (lane % 32): its half lane / 32 owns 16 consecutive
// tokens of each 32, score i is token 16 (lane / 32) + i, and scores 8 s .. 8 s + 7 are the
// second product's operand at step s as they stand.
//
// Bound by the VALU and the matrix cores together (per 32 rows x 64 tokens a wave has 32 MFMAs
// of 32 clocks and about 390 other instructions, a third of them the conversions; counters show
// the VALU busy 66 % and the matrix cores 37 % of the time): two times 4096 rows of 16 heads on
// 8192 tokens 311 to 323 us, 0.9 PFLOP/s, 8192 rows of 32 heads 594 us, 0.93. Looking for weights
// that one float16 does not hold takes 4 % of it (9 % at 64 columns). Codes converted once for the workgroup and kept in 16
// bits double what the waves read from LDS, and lose (367 us against 341).
//
// LDS rows hold 16-byte chunks permuted by xor, so that eight lanes of a read fall into
// different banks: K rows (a token each) with bits 0, 1 and 4 of the token, V rows (a column
// each, 64 tokens) with bits 2 and 3 of the column.
template <int DP>
__device__ __forceinline__ int k_swizzle(int token) {
  const int f = DP >= 128 ? (token & 3) | ((token >> 2) & 4) : ((token >> 3) & 2) | (token & 1);
  return 16 * f;
}

template <int DT>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == CP_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

constexpr int kManyRows = 128;

template <class F>
__device__ __forceinline__ void unrolled2(F f) {
  f(std::integral_constant<int, 0>{});
  f(std::integral_constant<int, 1>{});
}

template <int DT, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void attn_many_kernel(AttnArgs a, KvBatch bt, int items) {
  constexpr int NC = DP / 32, NL = DP / 64;          // 32-column chunks; direct loads of a wave for K, and for V
  constexpr int KB = kTile * DP, BUF = 2 * KB;       // bytes of a K (or V) tile, of a buffer
  extern __shared__ __align__(16) uint8_t lds[];     // [3][BUF], then [4 waves][NC][64 lanes][16]
  const KvCacheArgs& c = a.c;
  const int h = (int)(blockIdx.x % c.heads);
  const int split = (int)(blockIdx.x / c.heads % a.splits);
  int b, item, n_b;
  int64_t row0;
  // last items first: causal rows at the end of a prompt see the most tokens
  const int from_end = items - 1 - (int)(blockIdx.x / c.heads / a.splits), piece = h * a.splits + split;
  if (!kv_locate(bt, from_end, [&](int, int n) { return (int)(((int64_t)n * a.group + kManyRows - 1) / kManyRows); }, &b,
                 &item, &row0, &n_b))
    return attn_unowned<DT>(a, bt, item, items - from_end + item, piece, 0, 0);
  if (row0 < 0 || row0 + n_b > a.rows) {
    if (item == 0) attn_unowned<DT>(a, bt, -1, 0, piece, row0, n_b);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane & 31, hh = lane >> 5;
  const int d = c.d, blk = c.block, lb = 31 - __clz(c.block);
  const int len = max(__builtin_amdgcn_readfirstlane(a.lens[b]), 0);
  const int held = (int)min((int64_t)len, (int64_t)c.max_pages * blk);  // by the table

  // token range [lo, hi) of row r of the sequence; rows past the end see nothing
  auto range = [&](int64_t r, int* lo, int* hi) {
    const bool real = r < (int64_t)n_b * a.group;
    const int64_t pos = (int64_t)len - n_b + r / a.group;
    *hi = real ? (a.causal ? (int)max((int64_t)0, min((int64_t)held, pos + 1)) : held) : 0;
    *lo = a.window > 0 ? (int)max((int64_t)0, pos - a.window + 1) : 0;
    if (*lo >= *hi) *lo = *hi = 0;
  };
  const int64_t r0 = (int64_t)item * kManyRows, r = r0 + 32 * wave + q;
  int lo, hi;
  range(r, &lo, &hi);
  // what the workgroup's rows see together: rows are in order of position, so the first row
  // that sees anything bounds it below and the last one above
  int jlo, jhi;
  {
    int64_t last = min(r0 + kManyRows, (int64_t)n_b * a.group) - 1;
    // a row more than the window past the tokens held sees none of them
    if (a.window > 0) last = max(r0, min(last, ((int64_t)held + a.window - 1 - len + n_b) * a.group - 1));
    int x;
    range(last, &x, &jhi);
    // the lowest token of the first row whose position is not negative
    const int64_t first = max(r0, (int64_t)(n_b - len) * a.group);
    range(min(first, last), &jlo, &x);
    if (jhi == 0) jlo = 0;
  }
  // every real row of this wave sees all of a tile inside [wlo, whi)
  int wlo = lo, whi = hi;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    wlo = max(wlo, __shfl_xor(wlo, s));
    whi = min(whi, __shfl_xor(whi, s));
  }
  wlo = __builtin_amdgcn_readfirstlane(wlo);
  whi = __builtin_amdgcn_readfirstlane(whi);
  const int t0 = jlo / kTile, nt = (jhi + kTile - 1) / kTile - t0;
  const int per = max((nt + a.splits - 1) / a.splits, a.least), used = (nt + per - 1) / per;
  if (split > 0 && split >= used) return;
  const int tb = t0 + split * per, te = min(t0 + nt, tb + per);

  u32x4 qf[NC][2];
  const int64_t qrow = row0 + r / a.group;
  const int qh = h * a.group + (int)(r % a.group);
  const bool real = r < (int64_t)n_b * a.group;
  {
    typedef typename Elem<DT>::T T;
    const T* qp = (const T*)a.q + (real ? qrow * a.q_row + (int64_t)qh * a.q_head : 0);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const bool in = real && 32 * k + 16 * hh < d;
      const u32x4 z = {0, 0, 0, 0};
      qf[k][0] = in ? *reinterpret_cast<const u32x4*>(qp + 32 * k + 16 * hh) : z;
      qf[k][1] = in ? *reinterpret_cast<const u32x4*>(qp + 32 * k + 16 * hh + 8) : z;
    }
  }
  f32x16 o[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.0f;
  float m = kNegInf, l = 0.0f;

  const int* tab = c.table + (int64_t)b * c.max_pages;
  // direct loads. K: rows 1024 / DP each, all in the wave's 16-token group. V: 16 columns
  // each, four token groups. Chunks past d repeat the row's first, rows past d its last 16
  // (their q is 0, their results are dropped).
  // What changes from tile to tile is a page's start and where in the page the tile begins:
  // j0 is a multiple of 64 and a page's length a power of two, so (j0 + x) mod block is the sum
  // of the two parts' remainders for x < 64.
  constexpr int CH = DP / 16;
  const uint32_t page = (uint32_t)c.heads * blk * d;          // at most 65535 * 128 * 256
  const int kt = 16 * wave + lane / CH;                       // + 1024 / DP per load
  const int vg = (lane & 3) ^ ((lane >> 4) & 3);
  const uint8_t* const kbase = c.k + (int64_t)h * blk * d;
  const uint8_t* const vbase = c.v + (int64_t)h * blk * d;
  uint32_t koff[NL], voff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int token = kt + i * (1024 / DP);
    const int col = (16 * (lane % CH)) ^ k_swizzle<DP>(token);
    koff[i] = (token & (blk - 1)) * d + (col < d ? col : 0);
    voff[i] = min(16 * (wave * NL + i) + (lane >> 2), d - 1) * blk + ((16 * vg) & (blk - 1));
  }
  auto fetch = [&](int into, int tile, int pk, int pv) {
    uint8_t* to = lds + into * BUF;
    const int in = (tile * kTile) & (blk - 1);
    // no page: page 0's codes, which no row sees; K's page is the wave's
    pk = __builtin_amdgcn_readfirstlane(pk);
    const uint8_t* kp = kbase + (uint64_t)((unsigned)pk < (unsigned)c.pages ? pk : 0) * page + in * d;
    const uint8_t* vp = vbase + in + (uint64_t)((unsigned)pv < (unsigned)c.pages ? (unsigned)pv : 0u) * page;
#pragma unroll
    for (int i = 0; i < NL; ++i)
      __builtin_amdgcn_global_load_lds((gptr_t)(kp + koff[i]), (lptr_t)(to + (wave * NL + i) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < NL; ++i)
      __builtin_amdgcn_global_load_lds((gptr_t)(vp + voff[i]), (lptr_t)(to + KB + (wave * NL + i) * 1024), 16, 0, 0);
  };
  // this lane's K rows and V columns in LDS
  const int token = 16 * ((q >> 2) & 1) + 4 * (q >> 3) + (q & 3);
  const int ksw = k_swizzle<DP>(token);
  const int vsw = 16 * ((q >> 2) & 3);

  // Page numbers are looked up two tiles ahead and scales loaded one ahead. The compiler waits
  // for all loads in flight at a tile's end, where it moves these to the next tile's names: half
  // a tile after they, and the direct loads with them, were issued. Lookups past the last token repeat its own; such tokens are not seen.
  const int lastj = max(jhi - 1, 0);
  struct Pages {
    int k, v, g[2];
  } pn;
  auto at = [&](int j) {  // 32-bit offsets: max_pages is at most 2^31 / 128
    return *reinterpret_cast<const int*>(reinterpret_cast<const char*>(tab) + 4 * ((uint32_t)min(j, lastj) >> lb));
  };
  auto lookup = [&](int tile) {
    const int j0 = tile * kTile;
    pn.k = at(j0 + 16 * wave);
    pn.v = at(j0 + 16 * vg);
#pragma unroll
    for (int s = 0; s < 2; ++s) pn.g[s] = at(j0 + 32 * s + 16 * hh);
  };
  float ks[2], vs[2], nks[2], nvs[2];
  bool have[2], nhave[2];
  auto next_scales = [&](const int (&pg)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      nhave[s] = (unsigned)pg[s] < (unsigned)c.pages;
      const uint64_t hv = (uint64_t)(nhave[s] ? (unsigned)pg[s] : 0u) * (uint32_t)(4 * c.heads);
      nks[s] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(c.k_scale + h) + hv);
      nvs[s] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(c.v_scale + h) + hv);
    }
  };
  // A tile is two units of 32 tokens. A unit's scores are multiplied while the weights of the
  // unit before it are computed, so that the matrix cores and the VALU overlap within a wave.
  f32x16 sc[2];
  u32x4 kr[NC], vr[NC];
  auto read_k = [&](int buf, int s, int k) {
    kr[k] = *reinterpret_cast<const u32x4*>(lds + buf * BUF + token * DP + s * 32 * DP + ((32 * k + 16 * hh) ^ ksw));
  };
  auto read_v = [&](int buf, int s, int i) {
    vr[i] = *reinterpret_cast<const u32x4*>(lds + buf * BUF + KB + q * 64 + i * 32 * 64 + ((32 * s + 16 * hh) ^ vsw));
  };
  // the largest and least raw scores of the unit at hand (this lane's half of its row)
  float top = kNegInf, bot = -kNegInf;
  uint64_t marked[NC > 4 ? 2 : 1] = {};  // bit 16 i + j (of a word for four i): result (i, j) has seen a NaN code
  int buf = 0, nbuf = 1;                 // buffers of this tile and the next
  int pg[2] = {0, 0};  // pages of the next tile's scales
  if (tb < te) {
    lookup(tb);
    fetch(0, tb, pn.k, pn.v);
    next_scales(pn.g);
    lookup(tb + 1);
    fetch(1, tb + 1, pn.k, pn.v);
    pg[0] = pn.g[0], pg[1] = pn.g[1];
    lookup(tb + 2);
    __syncthreads();
  }
  // masks the scores of unit s of the tile at j0, of which the row may not see every token
  auto mask = [&](f32x16& x, int j0, int s, bool hv) {
    // this lane's first token, hidden from the compiler: it would compare all of them on
    // every tile, ahead of the branch
    int j1 = j0 + 32 * s + 16 * hh;
    asm volatile("" : "+v"(j1));
    top = kNegInf, bot = -kNegInf;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool see = hv && j1 + i >= lo && j1 + i < hi;
      bot = fminf(bot, see ? x[i] : -kNegInf);
      x[i] = see ? x[i] : kNegInf;
      top = fmaxf(top, x[i]);
    }
  };
  // As in attn_few_kernel: V's NaN codes of that unit leave the product and return to the rows
  // that see them, in a loop over the wave's LDS that costs the common path no registers.
  u32x4* const mine = reinterpret_cast<u32x4*>(lds + 3 * BUF) + wave * NC * 64 + lane;
  auto take_nan = [&](int j0, int s, bool hv) {
    u32x4 one[2];
    int j1 = j0 + 32 * s + 16 * hh;
    asm volatile("" : "+v"(j1));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int j = j1 + 2 * k;
      one[k >> 2][k & 3] = (hv && j >= lo && j < hi ? 0x3C00u : 0u) | (hv && j + 1 >= lo && j + 1 < hi ? 0x3C000000u : 0u);
    }
#pragma unroll
    for (int i0 = 0; i0 < NC; i0 += 4) {
#pragma clang loop unroll(disable)
      for (int i = i0; i < min(NC, i0 + 4); ++i) {
        u32x4 x = mine[64 * i], f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t fl = nan_flags(x[k]) >> 7;
          x[k] &= ~(fl * 0xFFu);
          f[k] = fl * 0x38u;  // 1.0 where the code was NaN
        }
        mine[64 * i] = x;
        f32x16 cnt;
#pragma unroll
        for (int j = 0; j < 16; ++j) cnt[j] = 0.0f;
        cnt = mfma32<CP_F16>(codes_to_16<CP_F16>(f[0], f[1]), one[0], cnt);
        cnt = mfma32<CP_F16>(codes_to_16<CP_F16>(f[2], f[3]), one[1], cnt);
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) bits |= cnt[j] > 0.0f ? 1u << j : 0;
        marked[i0 >> 2] |= (uint64_t)bits << (16 * (i - i0));
      }
    }
  };
  // the running maximum and what hangs on it, when a row's t passes it by kLag; called seldom
  auto move_max = [&](float tm) {
    tm = fmaxf(tm, __shfl_xor(tm, 32));
    const float mn = fmaxf(m, tm), ah = half_move(m, mn), al = ah * ah;
    m = mn;
    l = l * ah * ah;
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] *= al;
  };
  int tile = tb, last = 0;
  int wide = -1;  // the unit of the tile at hand from which on weights take two terms; -1: none does
  bool all, edge;
  auto enter = [&] {  // the tile at hand
    const int j0 = tile * kTile;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      have[s] = nhave[s];
      ks[s] = have[s] ? nks[s] : 1.0f, vs[s] = have[s] ? nvs[s] : 1.0f;  // as in attn_few_kernel
    }
    all = !__any(!have[0] || !have[1]);
    edge = !all || j0 < wlo || j0 + kTile > whi;
    last = nbuf == 2 ? 0 : nbuf + 1;  // the tile before this one's: the one after the next's
  };
  auto advance = [&] {  // ahead of a tile's second unit
    __syncthreads();    // the next tile has landed, and every wave is done with the one before this
    next_scales(pg);
    pg[0] = pn.g[0], pg[1] = pn.g[1];
    fetch(last, tile + 2, pn.k, pn.v);  // past the end: some page's codes, never used
    lookup(tile + 3);
  };
  if (tb < te) enter();
  while (tile < te) {
#pragma unroll
    for (int k = 0; k < NC; ++k) read_k(buf, 0, k);
#pragma unroll
    for (int j = 0; j < 16; ++j) sc[0][j] = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      sc[0] = mfma32<DT>(codes_to_16<DT>(kr[k][0], kr[k][1]), qf[k][0], sc[0]);
      sc[0] = mfma32<DT>(codes_to_16<DT>(kr[k][2], kr[k][3]), qf[k][1], sc[0]);
    }
    top = bot = sc[0][0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, sc[0][j]), bot = fminf(bot, sc[0][j]);
    wide = -1;
    while (tile < te) {
      const int j0 = tile * kTile;
      unrolled2([&](auto S) {
        constexpr int s = S;
        if (s == 1 && wide >= 0) return;
        const float kc = ks[s] * a.scale;
        const float lg = (float)((int)(__float_as_uint(vs[s]) >> 23) - 127);
        const float iv = __uint_as_float((254u << 23) - (__float_as_uint(vs[s]) & 0x7F800000u));
        if constexpr (s == 1) advance();
#pragma unroll
        for (int k = 0; k < NC; ++k) read_k(s ? nbuf : buf, 1 - s, k);
        if (edge) mask(sc[s], j0, s, have[s]);
        // the largest t of the unit: kc > 0, so t rises with the raw score
        const float tm = __builtin_fmaf(top, kc, lg);
        if (__any(tm > m + kLag)) move_max(tm);
        if (__any(__builtin_fmaf(bot, kc, lg) < m - kDeep)) {
          wide = s;
          return;
        }
        const float off = lg + kLift - (m == kNegInf ? 0.0f : m);
        // one MFMA of the next unit's scores, then as many of this unit's weights as it covers
        u32x4 w[2];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[1 - s][j] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * NC; ++k) {
          const u32x4 x = kr[k >> 1];
          sc[1 - s] = mfma32<DT>(k & 1 ? codes_to_16<DT>(x[2], x[3]) : codes_to_16<DT>(x[0], x[1]), qf[k >> 1][k & 1],
                                 sc[1 - s]);
#pragma unroll
          for (int i = 8 * k / (2 * NC); i < 8 * (k + 1) / (2 * NC); ++i) {
            const float e0 = exp2_fast(__builtin_fmaf(sc[s][2 * i], kc, off));
            const float e1 = exp2_fast(__builtin_fmaf(sc[s][2 * i + 1], kc, off));
            sum += e0 + e1;
            uint32_t e = pack2<CP_F16>(e0, e1);
            asm volatile("" : "+v"(e));  // here, not past the branch below
            w[i >> 2][i & 3] = e;
          }
          if (k == NC) {
#pragma unroll
            for (int i = 0; i < NC; ++i) read_v(buf, s, i);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        l = __builtin_fmaf(sum, iv, l);
        if (edge) {
          uint32_t any = 0;
#pragma unroll
          for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) any |= nan_flags(vr[i][k]);
          if (__any(any != 0)) {
#pragma unroll
            for (int i = 0; i < NC; ++i) mine[64 * i] = vr[i];
            take_nan(j0, s, have[s]);
#pragma unroll
            for (int i = 0; i < NC; ++i) vr[i] = mine[64 * i];
          }
        }
        // The second product, and the next unit's largest and least scores beside it. It gives way to the
        // SIMD's other wave: its MFMAs need an issue slot in 32 clocks, the weights every slot, and
        // two waves that keep out of step overlap (335 -> 309 us for two prompts of 4096 rows).
        __builtin_amdgcn_s_setprio(0);
        top = bot = sc[1 - s][0];
#pragma unroll
        for (int k = 0; k < 2 * NC; ++k) {
          const int i = k % NC;
          const u32x4 x = vr[i];
          o[i] = mfma32<CP_F16>(k < NC ? codes_to_16<CP_F16>(x[0], x[1]) : codes_to_16<CP_F16>(x[2], x[3]), w[k / NC], o[i]);
#pragma unroll
          for (int j = 16 * k / (2 * NC); j < 16 * (k + 1) / (2 * NC); ++j)
            top = fmaxf(top, sc[1 - s][j]), bot = fminf(bot, sc[1 - s][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(1);
      });
      if (wide >= 0) break;
      buf = nbuf;
      nbuf = last;
      ++tile;
      enter();
    }
    // Weights in two terms, a unit at a time from its scores on, until a tile needs no more of
    // them. Every tile has its one barrier in either loop, so waves of both kinds keep in step.
    // Two prompts of 4096 rows whose scores' deviation is 5.5 (all units here) 495 us, 1.4 (a few) 331.
    bool deep = true;  // the tile at hand needs them
    for (bool ahead = wide == 1; tile < te;) {
      const int s = wide, j0 = tile * kTile;
      if (s == 1 && !ahead) advance();
      ahead = false;
      const bool hv = s ? have[1] : have[0];
      const float v1 = s ? vs[1] : vs[0], kc = (s ? ks[1] : ks[0]) * a.scale;
      const float lg = (float)((int)(__float_as_uint(v1) >> 23) - 127);
      f32x16& x = sc[0];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = 0.0f;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        read_k(buf, s, k);
        x = mfma32<DT>(codes_to_16<DT>(kr[k][0], kr[k][1]), qf[k][0], x);
        x = mfma32<DT>(codes_to_16<DT>(kr[k][2], kr[k][3]), qf[k][1], x);
      }
      if (edge) {
        mask(x, j0, s, hv);
      } else {
        top = bot = x[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) top = fmaxf(top, x[j]), bot = fminf(bot, x[j]);
      }
      const float tm = __builtin_fmaf(top, kc, lg);
      if (__any(tm > m + kLag)) move_max(tm);
      deep |= __any(__builtin_fmaf(bot, kc, lg) < m - kDeep);
      // as in attn_few_kernel, the sum's terms and the weights from them
      const float off = kLift - (m == kNegInf ? 0.0f : m);
      u32x4 wh[2], wl[2];
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e0 = exp2_fast(__builtin_fmaf(x[2 * i], kc, off)), e1 = exp2_fast(__builtin_fmaf(x[2 * i + 1], kc, off));
        sum += e0 + e1;
        const Weights2 w = weights2(e0 * v1, e1 * v1);
        wh[i >> 2][i & 3] = w.hi, wl[i >> 2][i & 3] = w.lo;
      }
      l += sum;
#pragma unroll
      for (int i = 0; i < NC; ++i) read_v(buf, s, i);
      if (edge) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) any |= nan_flags(vr[i][k]);
        if (__any(any != 0)) {
#pragma unroll
          for (int i = 0; i < NC; ++i) mine[64 * i] = vr[i];
          take_nan(j0, s, hv);
#pragma unroll
          for (int i = 0; i < NC; ++i) vr[i] = mine[64 * i];
        }
      }
#pragma unroll
      for (int k = 0; k < 2 * NC; ++k) {
        const int i = k % NC;
        const u32x4 y = vr[i], c16 = k < NC ? codes_to_16<CP_BF16>(y[0], y[1]) : codes_to_16<CP_BF16>(y[2], y[3]);
        o[i] = mfma32<CP_BF16>(c16, wh[k / NC], o[i]);
        o[i] = mfma32<CP_BF16>(c16, wl[k / NC], o[i]);
      }
      wide = 1 - s;
      if (s == 1) {
        buf = nbuf;
        nbuf = last;
        ++tile;
        enter();
        if (!deep) break;
        deep = false;
      }
    }
  }
  __syncthreads();  // the last fetch is in before LDS is given up
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (__any(marked[i >> 2] != 0)) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        o[i][j] = marked[i >> 2] >> (16 * (i & 3) + j) & 1 ? __builtin_nanf("") : o[i][j];
    }
  }
  l += __shfl_xor(l, 32);
  if (!real) return;
  const int64_t orow = qrow * ((int64_t)a.group * c.heads) + qh;
  // lane's results: columns 32 i + 8 (j / 4) + 4 hh + j % 4 of its row
  const SplitParts sp = split_parts(a);
  if (a.splits > 1 && split == 0 && hh == 0) sp.used[orow] = used > 1 ? used : 0;
  if (used > 1) {
    float* p = sp.sums + (orow * a.splits + split) * d;
    float* pm = sp.ml + (orow * a.splits + split) * 2;
    if (hh == 0) pm[0] = m, pm[1] = l;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = 32 * i + 8 * j + 4 * hh;
        if (x < d) *reinterpret_cast<f32x4*>(p + x) = f32x4{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
      }
    return;
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  typename Elem<DT>::T* op = (typename Elem<DT>::T*)a.out + orow * d;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int x = 32 * i + 8 * j + 4 * hh;
      u32x2 v;
      v[0] = pack2<DT>(o[i][4 * j] * inv, o[i][4 * j + 1] * inv);
      v[1] = pack2<DT>(o[i][4 * j + 2] * inv, o[i][4 * j + 3] * inv);
      if (x < d) *reinterpret_cast<u32x2*>(op + x) = v;
    }
  if (a.lse && hh == 0) a.lse[orow] = row_lse(m, l);
}

// The splits of a row joined, in a fixed order. Bound by latency, or by reading the splits'
// sums. d / 4 threads (a group) take a row's columns; with more than eight splits the groups
// of a workgroup share one row's, otherwise each has its own row (attention and join, one row
// of 16 heads: on 32768 tokens in 64 splits 27.7 us a group a row, 19.5 a workgroup; on 64 x
// 2048 in two 25.8 and 26.5).
template <int DT, bool ONE_ROW>
__global__ __launch_bounds__(256) void attn_join_kernel(SplitParts sp, int64_t rows, int d, int most,
                                                        typename Elem<DT>::T* __restrict__ out,
                                                        float* __restrict__ lse) {
  __shared__ float sm_m[4], sm_l[16];
  __shared__ __align__(16) float sm_o[256 * 4];
  const int T = d / 4, NG = min(256 / T, 16), grp = threadIdx.x / T, c = 4 * (threadIdx.x % T);
  const int64_t row = ONE_ROW ? blockIdx.x : (int64_t)blockIdx.x * NG + grp;
  const bool mine = grp < NG && row < rows;
  // bounded: offsets that decrease leave rows without a count
  const int splits = mine || ONE_ROW ? min(max(sp.used[row], 0), most) : 0;
  if (splits == 0) return;  // ONE_ROW: the whole workgroup leaves
  const float* po = sp.sums + row * most * d;
  const float* pm = sp.ml + row * most * 2;
  float mm = kNegInf;
  if constexpr (ONE_ROW) {
    for (int s = threadIdx.x; s < splits; s += 256) mm = fmaxf(mm, pm[2 * s]);
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) mm = fmaxf(mm, __shfl_xor(mm, k));
    if ((threadIdx.x & 63) == 0) sm_m[threadIdx.x >> 6] = mm;
    __syncthreads();
    mm = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  } else {
    for (int s = 0; s < splits; ++s) mm = fmaxf(mm, pm[2 * s]);
  }
  const float ms = mm == kNegInf ? 0.0f : mm;
  f32x4 v = {0, 0, 0, 0};
  float ll = 0.0f;
  if (mine) {
#pragma unroll 4
    for (int s = ONE_ROW ? grp : 0; s < splits; s += ONE_ROW ? NG : 1) {
      const float fh = half_move(pm[2 * s], ms);
      ll += pm[2 * s + 1] * fh * fh;
      v += *reinterpret_cast<const f32x4*>(po + (int64_t)s * d + c) * (fh * fh);
    }
  }
  if constexpr (ONE_ROW) {
    if (mine) {
      *reinterpret_cast<f32x4*>(&sm_o[grp * d + c]) = v;
      sm_l[grp] = ll;  // the group's threads hold the same sum
    }
    __syncthreads();
    if (grp != 0) return;
    for (int i = 1; i < NG; ++i) {
      v += *reinterpret_cast<const f32x4*>(&sm_o[i * d + c]);
      ll += sm_l[i];
    }
  }
  const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
  u32x2 y;
  y[0] = pack2<DT>(v[0] * inv, v[1] * inv);
  y[1] = pack2<DT>(v[2] * inv, v[3] * inv);
  *reinterpret_cast<u32x2*>(out + row * d + c) = y;
  if (lse && c == 0) lse[row] = row_lse(mm, ll);
}

struct AttnPlan {
  bool many;
  int64_t items;  // upper bound of the batch's row tiles, and one more where rows may have no sequence
  int splits, least;  // at most so many pieces of a row's tiles, of at least so many tiles
};

// Row tiles of 16 while a sequence has up to 64 (row, head of the group) pairs on average, or
// while all pairs times the tokens they can see are few: four small workgroups a CU start and
// end faster, and what they read more often comes from the L2. Tiles of 128 above that, where
// the weights' arithmetic counts. Rows of 8 heads on 4 x 8192 tokens, tiles of 16 / of 128: 16
// rows 16 / 36 us, 64 25 / 50, 256 83 / 62; 16 heads, 1024 rows on as many tokens 22 / 30, 1024
// on 2048 44 / 41, 512 on 4096 50 / 41.
static AttnPlan attn_plan(int64_t rows, int64_t batch, bool ragged, int group, int heads, int d,
                          int64_t cap, int window) {
  AttnPlan p;
  p.many = rows * group > 64 * batch &&
           (double)rows * group * heads * (window > 0 ? std::min(cap, (int64_t)window + kManyRows) : cap) > 1 << 24;
  const int tile = p.many ? kManyRows : 16, step = p.many ? kTile : kFewTile;
  p.items = ragged ? rows * group / tile + batch : batch * ((group + tile - 1) / tile);
  const int64_t n = std::max(p.items * heads, (int64_t)1);
  const int64_t span = window > 0 ? std::min(cap, (int64_t)window + tile + step) : cap;
  int64_t s = 1;
  if (batch == 0) {
    // no sequence: the rows are cleared
  } else if (p.many) {
    // The tokens of a row tile are split as takes the fewest predicted microseconds. A join takes
    // a launch (4) and the time in which the splits' float32 outputs are written and read back.
    const int dp = d <= 64 ? 64 : d <= 128 ? 128 : 256;
    const double mb = (double)rows * group * heads * d * 8 / 1e6;  // those outputs, a split
    const int64_t tiles = (span + step - 1) / step;
    if (n < 128) {
      // CUs to spare: a tile takes 2.2 (at 128 columns) while no more workgroups run than fit at
      // once (two a CU), and tiles t / s + join j s are fewest at s = sqrt(t / j). 40 row tiles
      // on 32768 tokens: 674 us in one, 127 in six, 100 in eight, 92 in sixteen (99 as chosen).
      const double tile_us = 2.2 * dp / 128, join_us = mb / 4;
      const int64_t x = std::min({(dp > 128 ? 256 : 512) / n, tiles / 2, (int64_t)std::sqrt(tiles * tile_us / join_us)});
      if (x > 1 && (tiles + x - 1) / x * tile_us + x * join_us + 4.0 < tiles * tile_us) s = x;
    } else {
      // A CU or more for each: the tiles of all pieces at 1.6 a CU (two workgroups on one are
      // hardly faster than one after the other), and half a piece for the last to end, lengths
      // being ragged. 264 row tiles, 1000 rows each of two sequences up to 4096: 169 us in one,
      // 110 in two, 88 in three, 89 in four, 101 in six; 616, 2400 rows of two up to 8192: 359,
      // 280, 248, 268, 296; 520, 4096 rows of one on 8192: 255, 249, 261, 271, 296.
      const double cus = dp > 128 ? 128 : 256, tile_us = dp > 128 ? 3.2 : 1.6;
      double best = 0.0;
      for (int64_t x = 1; x == 1 || (x <= 4 && x <= tiles / 2); ++x) {
        const double us = (std::max(1.0, n * x / cus) + 0.5) * ((double)tiles / x + 1) * tile_us +
                          (x > 1 ? 4.0 + x * mb / 6 : 0.0);
        if (x == 1 || us < best) best = us, s = x;
      }
    }
  } else {
    // As many workgroups as the CUs hold at once, but pieces of no less than 8 steps of the
    // longest row tile there can be, or 4 of a shorter one's (16 and 8, then 4 and 4, for one row
    // of 16 heads on 4 x 1024 tokens 11.9, 9.8, 9.2 us, on 8192 12.9, 10.6, 11.0, on 300 7.5,
    // 7.5, 9.2).
    s = std::max((int64_t)1, std::min(1024 / n, span / (8 * step)));
  }
  p.items += ragged;
  p.least = p.many ? 2 : 4;
  p.splits = (int)s;
  return p;
}

template <int DT, int DP>
static int attn_launch(const AttnArgs& a, const KvBatch& b, const AttnPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.items * a.c.heads * a.splits));
  if (p.many) {
    constexpr int lds = 6 * kTile * DP + 4 * (DP / 32) * 1024;
    static std::atomic<uint64_t> done{0};
    if (int s = allow_lds(reinterpret_cast<const void*>(&attn_many_kernel<DT, DP>), lds, &done, "LDS of the cache attention"))
      return s;
    attn_many_kernel<DT, DP><<<grid, 256, lds, st>>>(a, b, (int)p.items);
  } else {
    attn_few_kernel<DT, DP><<<grid, 256, 0, st>>>(a, b, (int)p.items);
  }
  CP_LAUNCHED("cache attention");
  return CP_OK;
}

template <int DT>
static int attn_launch_d(const AttnArgs& a, const KvBatch& b, const AttnPlan& p, hipStream_t st) {
  const int s = a.c.d <= 64    ? attn_launch<DT, 64>(a, b, p, st)
                : a.c.d <= 128 ? attn_launch<DT, 128>(a, b, p, st)
                               : attn_launch<DT, 256>(a, b, p, st);
  if (s || a.splits == 1) return s;
  const int64_t n = a.rows * a.group * a.c.heads;
  typename Elem<DT>::T* out = (typename Elem<DT>::T*)a.out;
  const int64_t groups = std::min(256 / (a.c.d / 4), 16);
  if (a.splits > 8)
    attn_join_kernel<DT, true><<<dim3((unsigned)n), 256, 0, st>>>(split_parts(a), n, a.c.d, a.splits, out, a.lse);
  else
    attn_join_kernel<DT, false><<<dim3((unsigned)((n + groups - 1) / groups)), 256, 0, st>>>(split_parts(a), n, a.c.d,
                                                                                          a.splits, out, a.lse);
  CP_LAUNCHED("cache attention's join");
  return CP_OK;
}

static int attn_check(const cp_kv_cache* cache, int64_t rows, int q_heads, const int32_t* table,
                      int64_t batch, int64_t max_pages, const int32_t* offsets) {
  if (int s = kv_check_cache(cache)) return s;
  if (int s = kv_check_batch(table, batch, max_pages, rows, offsets)) return s;
  // pages are looked up, in 32 bits, up to three tiles past a sequence's last
  if (max_pages * cache->block > 0x7FFFFFFF - 1023)
    return set_error(CP_ERR_SHAPE, "table rows of %lld pages of %d tokens", (long long)max_pages, cache->block);
  if (q_heads < 1 || q_heads % cache->heads)
    return set_error(CP_ERR_SHAPE, "%d query heads over %d cache heads", q_heads, cache->heads);
  return CP_OK;
}

}  // namespace cp

extern "C" {

size_t cp_kv_attention_ws_bytes(const cp_kv_cache* cache, int64_t rows, int q_heads, int64_t batch,
                                int64_t max_pages, int ragged, int window) {
  if (!cache || cache->heads < 1 || rows < 1 || q_heads < 1 || batch < 0 || max_pages < 1) return 0;
  const cp::AttnPlan p = cp::attn_plan(rows, batch, ragged != 0, q_heads / cache->heads, cache->heads,
                                       cache->head_dim, max_pages * cache->block, window);
  return p.splits > 1 ? (size_t)rows * q_heads * p.splits * (cache->head_dim + 2) * 4 + (size_t)rows * q_heads * 4 : 0;
}

int cp_kv_attention(const cp_kv_cache* cache, const void* q, int64_t q_row, int64_t q_head, int dtype,
                    int64_t rows, int q_heads, const int32_t* table, int64_t batch, int64_t max_pages,
                    const int32_t* lens, const int32_t* offsets, int causal, int window, float scale,
                    void* out, float* lse, void* ws, size_t ws_bytes, void* stream) {
  cp::clear_error();
  if (int s = cp::attn_check(cache, rows, q_heads, table, batch, max_pages, offsets)) return s;
  if (dtype != CP_BF16 && dtype != CP_F16) return cp::set_error(CP_ERR_ARG, "queries are bfloat16 or float16");
  if (window < 0) return cp::set_error(CP_ERR_ARG, "window %d", window);
  if (!(scale > 0.0f) || !(scale < 3e38f)) return cp::set_error(CP_ERR_ARG, "scale %g must be positive", scale);
  if (rows == 0) return CP_OK;
  if (!q || (batch && !lens) || !out) return cp::set_error(CP_ERR_ARG, "null q / lens / out");
  if (!cp::aligned(q, 16) || q_row * 2 % 16 || q_head * 2 % 16 || !cp::aligned(out, 16))
    return cp::set_error(CP_ERR_ALIGN, "rows and heads of q and out need 16-byte alignment");
  if (q_row < 0 || q_head < 0) return cp::set_error(CP_ERR_SHAPE, "negative stride of q");
  const int group = q_heads / cache->heads;
  const cp::AttnPlan p = cp::attn_plan(rows, batch, offsets != nullptr, group, cache->heads, cache->head_dim,
                                       max_pages * cache->block, window);
  // a join takes up to a workgroup a row and head
  if (p.items * cache->heads * p.splits > cp::most_workgroups(256) || rows * q_heads > 0x7FFFFFFF ||
      (p.splits > 1 && rows * q_heads > cp::most_workgroups(256)))
    return cp::set_error(CP_ERR_SHAPE, "too many rows");
  const size_t need = cp_kv_attention_ws_bytes(cache, rows, q_heads, batch, max_pages, offsets != nullptr, window);
  if (need && (!ws || ws_bytes < need))
    return cp::set_error(CP_ERR_WORKSPACE, "workspace of %zu bytes needs %zu", ws_bytes, need);
  if (need && !cp::aligned(ws, 256)) return cp::set_error(CP_ERR_ALIGN, "workspace needs 256-byte alignment");
  cp::AttnArgs a;
  a.c = cp::kv_args(cache, table, max_pages);
  a.q = q;
  a.q_row = q_row;
  a.q_head = q_head;
  a.lens = lens;
  a.out = out;
  a.lse = lse;
  a.part = (float*)ws;
  a.rows = rows;
  a.group = group;
  a.causal = causal != 0;
  a.window = window;
  a.splits = p.splits;
  a.least = p.least;
  a.scale = scale * cp::kLog2e;
  const cp::KvBatch b = {offsets, (int)batch};
  return dtype == CP_BF16 ? cp::attn_launch_d<CP_BF16>(a, b, p, (hipStream_t)stream)
                          : cp::attn_launch_d<CP_F16>(a, b, p, (hipStream_t)stream);
}

}  // extern "C"
