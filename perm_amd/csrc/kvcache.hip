// A paged key / value cache held in e4m3 with one power-of-two scale per page and head
// (gfx950): quantising rows as they are written, and reading them back.
//
// A page is `block` tokens (16, 32, 64 or 128) of every head. K codes lie [page][head]
// [block][d], V codes transposed, [page][head][d][block]: attention's second product sums
// over tokens, and its operand wants consecutive tokens of one column. k_scale and v_scale
// are [page][head] float32, 2^e with the least e in [-60, 60] that holds the page's largest
// finite magnitude: max |x| <= 448 * 2^e. A code is RNE to e4m3 of x * 2^-e, saturating at
// +-448; NaN stays NaN.
//
// Rows appended to a page begun earlier may need a larger scale. The codes held are then
// multiplied by 2^(old e - new e) and rounded again, which is exact but where a code falls
// into e4m3's subnormals: powers of two are what keeps repeated appends from eroding codes.
// Slots that no row is written to keep their codes.
#include <hip/hip_runtime.h>

#include "cp_device.h"
#include "kvcache.h"
#include "lowbit.h"

namespace cp {

// 2^e: the least e in [-60, 60] with a <= 448 * 2^e (448 = 0.875 * 2^9).
__device__ __forceinline__ float kv_scale(float a) {
  int e = a == 0.0f ? -60 : frexp_e(a) - 8 - (frexp_m(a) <= 0.875f ? 1 : 0);
  e = e < -60 ? -60 : e > 60 ? 60 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// 1 / 2^e, exactly.
__device__ __forceinline__ float inv_pow2(float s) {
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

__device__ __forceinline__ float kv_clamp(float v) {
  return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}

// Largest of v over the wave (all lanes active): within 16 lanes on the VALU, then across.
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<kDppXor1>(v));
  v = fmaxf(v, dpp<kDppXor2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  v = fmaxf(v, dpp<kDppRor8>(v));
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

struct KvRows {
  const void* p;            // [rows][head][d]
  int64_t row_st, head_st;  // element strides
};

// The largest finite magnitude of eight values.
__device__ __forceinline__ float amax8(const float (&v)[8], float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(v[i]);
    m = a < __builtin_inff() && a > m ? a : m;
  }
  return m;
}

__device__ __forceinline__ u32x2 codes8(const float (&v)[8], float inv) {
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = kv_clamp(v[i] * inv);
  return e4m3_encode8(u);
}

// Four codes times ratio, rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t c, float ratio) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, w, true);
}

// The low n bytes of a dword (none for n <= 0, all for n >= 4).
__device__ __forceinline__ uint32_t low_bytes(int n) {
  return n <= 0 ? 0u : n >= 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
}

// A 16-token slab of V passes through LDS as dwords of four columns, [d / 4][16 tokens] at
// this pitch in dwords: rows stay 16-byte aligned and neighbouring rows 20 banks apart.
constexpr int kSlabPitch = 20;
constexpr int kSlabLds = 256 / 4 * kSlabPitch;  // dwords of a wave

// Four dwords of four bytes, transposed: out[i] byte j = in[j] byte i.
__device__ __forceinline__ void transpose4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u), e = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(e, b, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(e, b, 0x07060302u);
}

// One wave per (touched page, head), so nothing waits for another wave. It takes the page's
// scales from the rows that fall into it, moves the codes held to a larger scale where it has
// to, and writes the rows' codes: K as they come, V transposed through LDS a slab of 16
// tokens at a time. Bound by HBM for prompts (17 000 tokens of 8 heads of 128 in bf16: 105 MB
// in 24 us, 4.4 TB/s), by latency for single tokens (64 sequences 7.8 us: length, page number,
// scale and codes are read one after the other).
//
// KEEP: pages of 16 tokens and d up to 128, whose values stay in registers between the scale
// and the codes; larger ones are read twice, the second time from the L2 (those prompts in pages of
// 32, 64 and 128 tokens 36, 41 and 50 us, a wave having the more to do the larger its page is).
template <int DT, bool KEEP>
__global__ __launch_bounds__(256, KEEP ? 4 : 3) void kv_write_kernel(KvCacheArgs c, KvRows k, KvRows v, KvBatch q, int64_t rows,
                                                       const int* filled) {
  __shared__ __align__(16) uint32_t slabs[4][kSlabLds];
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t* slab = slabs[wave];
  const int at = (int)blockIdx.x * 4 + wave, h = at % c.heads;
  int b, item, n_b;
  int64_t row0;
  if (!kv_locate(
          q, at / c.heads,
          [&](int s, int n) { return n ? (max(filled[s], 0) % c.block + n + c.block - 1) / c.block : 0; }, &b, &item,
          &row0, &n_b))
    return;
  const int held = max(filled[b], 0);
  const int64_t pg = (int64_t)held / c.block + item;                 // page of the sequence
  const int s0 = item == 0 ? held % c.block : 0;                     // first slot written
  const int done = item == 0 ? 0 : item * c.block - held % c.block;  // rows in earlier pages
  const int n = min(n_b - done, c.block - s0);
  const int64_t r0 = row0 + done;
  if (pg >= c.max_pages || r0 < 0 || r0 + n > rows) return;
  const int page = c.table[(int64_t)b * c.max_pages + pg];
  if ((unsigned)page >= (unsigned)c.pages) return;
  const int64_t ph = (int64_t)page * c.heads + h;
  const int d = c.d, blk = c.block, dc = d / 8, total = n * dc;
  uint8_t* kc = c.k + ph * blk * d;
  uint8_t* vc = c.v + ph * blk * d;
  const T* kp = (const T*)k.p + r0 * k.row_st + h * k.head_st;
  const T* vp = (const T*)v.p + r0 * v.row_st + h * v.head_st;

  // asked for before they are needed: the scales of the codes held, and (KEEP) the codes of V
  const float ko = c.k_scale[ph], vo = c.v_scale[ph];
  constexpr int CH = KEEP ? 4 : 1;
  Raw8<DT> kv[CH], vv[CH];
  float ka = 0.0f, va = 0.0f;
  if constexpr (KEEP) {
    // lanes past the rows repeat the last one's values, which changes no maximum
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int i = min(lane + 64 * u, total - 1), row = i / dc, col = 8 * (i - row * dc);
      kv[u] = load_raw8<DT>(kp + row * k.row_st + col);
      vv[u] = load_raw8<DT>(vp + row * v.row_st + col);
    }
  }
  u32x4 old[4];
  const bool partial = KEEP && n < 16;
  if (partial && lane < d / 4) {
#pragma unroll
    for (int y = 0; y < 4; ++y) old[y] = *reinterpret_cast<const u32x4*>(vc + (4 * lane + y) * blk);
  }
  float f[8];
  if constexpr (KEEP) {
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      widen8<DT>(kv[u], f);
      ka = amax8(f, ka);
      widen8<DT>(vv[u], f);
      va = amax8(f, va);
    }
  } else {
#pragma unroll 4
    for (int i = lane; i < total; i += 64) {
      const int row = i / dc, col = 8 * (i - row * dc);
      load8<DT>(kp + row * k.row_st + col, f);
      ka = amax8(f, ka);
      load8<DT>(vp + row * v.row_st + col, f);
      va = amax8(f, va);
    }
  }
  float ks = kv_scale(wave_max(ka)), vs = kv_scale(wave_max(va)), vratio = 1.0f;
  if (s0 > 0) {  // codes held: keep the larger scale
    if (ks > ko) {
      const float ratio = ko * inv_pow2(ks);
      for (int i = lane; i < s0 * d / 4; i += 64) {
        uint32_t* p = reinterpret_cast<uint32_t*>(kc) + i;
        *p = rescale4(*p, ratio);
      }
    } else {
      ks = ko;
    }
    if (vs > vo) vratio = vo * inv_pow2(vs);
    else vs = vo;
  }
  if (lane == 0) {
    c.k_scale[ph] = ks;
    c.v_scale[ph] = vs;
  }
  const float ki = inv_pow2(ks), vi = inv_pow2(vs);
  // slabs with a row written, and, where codes move, the ones before
  const int g0 = vratio != 1.0f ? 0 : s0 / 16, g1 = (s0 + n + 15) / 16;
  for (int g = g0; g < g1; ++g) {
    const int lo = max(s0 - 16 * g, 0), hi = min(s0 + n - 16 * g, 16);  // slots of the slab written
    // rows of this slab: lo .. hi - 1, from row 16 g + lo - s0
    const int first = 16 * g + lo - s0, cnt = max(hi - lo, 0) * dc;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (KEEP && u >= CH) break;
      const int i = lane + 64 * u;
      if (i >= cnt) break;
      const int row = i / dc, cc = i - row * dc;
      if constexpr (!KEEP) {
        kv[0] = load_raw8<DT>(kp + (first + row) * k.row_st + 8 * cc);
        vv[0] = load_raw8<DT>(vp + (first + row) * v.row_st + 8 * cc);
      }
      widen8<DT>(kv[KEEP ? u : 0], f);
      *reinterpret_cast<u32x2*>(kc + (int64_t)(16 * g + lo + row) * d + 8 * cc) = codes8(f, ki);
      widen8<DT>(vv[KEEP ? u : 0], f);
      const u32x2 w = codes8(f, vi);
      slab[2 * cc * kSlabPitch + lo + row] = w[0];
      slab[(2 * cc + 1) * kSlabPitch + lo + row] = w[1];
    }
    __builtin_amdgcn_wave_barrier();
    // four columns a lane: 16 tokens of each
    if (lane < d / 4) {
      uint8_t* out = vc + (int64_t)(4 * lane) * blk + 16 * g;
      u32x4 w[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const u32x4 r = *reinterpret_cast<const u32x4*>(slab + lane * kSlabPitch + 4 * x);
        const uint32_t in[4] = {r[0], r[1], r[2], r[3]};
        uint32_t t[4];
        transpose4(in, t);
#pragma unroll
        for (int y = 0; y < 4; ++y) w[y][x] = t[y];
      }
      if (lo > 0 || hi < 16) {  // the other slots keep their codes, the held ones moved
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if constexpr (!KEEP) old[y] = *reinterpret_cast<const u32x4*>(out + y * blk);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            // bytes written, and bytes held before
            const uint32_t put = low_bytes(hi - 4 * x) & ~low_bytes(lo - 4 * x), move = low_bytes(s0 - 16 * g - 4 * x);
            uint32_t o = old[y][x];
            if (vratio != 1.0f) o = (o & ~move) | (rescale4(o, vratio) & move);
            w[y][x] = (o & ~put) | (w[y][x] & put);
          }
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) *reinterpret_cast<u32x4*>(out + y * blk) = w[y];
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// One wave per (16 tokens held, head): the codes' values in rows [total][head][d]. V's slab
// is transposed through LDS. Bound by HBM, two thirds of the bytes being written (45 000 tokens
// of 8 heads of 128 to bf16: 276 MB in 53 us, 5.2 TB/s, a copy's rate). All of a wave's loads
// are issued before the first is used, and five waves a SIMD keep enough of them in flight.
template <int DT>
__global__ __launch_bounds__(256, 5) void kv_read_kernel(KvCacheArgs c, KvBatch q, int items, int64_t total,
                                                      typename Elem<DT>::T* __restrict__ ko,
                                                      typename Elem<DT>::T* __restrict__ vo) {
  __shared__ __align__(16) uint32_t slabs[4][kSlabLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t* slab = slabs[wave];
  const int at = (int)blockIdx.x * 4 + wave, h = at % c.heads;
  int b, item, n_b;
  int64_t row0;
  if (!kv_locate(q, at / c.heads, [&](int, int n) { return (n + 15) / 16; }, &b, &item, &row0, &n_b)) {
    // the rows that no sequence has, a (row, head) a lane, shared by the waves past the end
    if (at >= items * c.heads) return;
    const KvUnowned u = kv_unowned(q, total);
    const int64_t lead = u.lead * c.heads, skip = u.tail * c.heads - lead;
    const int64_t waves = (int64_t)(items - at / c.heads + item) * c.heads;
    for (int64_t i = ((int64_t)item * c.heads + h) * 64 + lane; i < total * c.heads - skip; i += waves * 64) {
      const int64_t to = (i < lead ? i : i + skip) * c.d;
      const float zero[8] = {};
      for (int x = 0; x < c.d; x += 8) {
        store8<DT>(ko + to + x, zero);
        store8<DT>(vo + to + x, zero);
      }
    }
    return;
  }
  const int64_t r0 = row0 + (int64_t)item * 16;
  if (r0 < 0) return;
  const int n = (int)min((int64_t)min(n_b - item * 16, 16), total - r0);  // rows that there are
  const int64_t pg = (int64_t)item * 16 / c.block;
  const int page = pg < c.max_pages ? c.table[(int64_t)b * c.max_pages + pg] : -1;
  const bool have = (unsigned)page < (unsigned)c.pages;
  const int64_t ph = have ? (int64_t)page * c.heads + h : 0;
  const int d = c.d, blk = c.block, dc = d / 8, slot = item * 16 % blk;
  const uint8_t* kc = c.k + ph * blk * d + slot * d;
  const uint8_t* vc = c.v + ph * blk * d + slot;
  const float ks = have ? c.k_scale[ph] : 0.0f, vs = have ? c.v_scale[ph] : 0.0f;
  u32x4 w[4];
  if (lane < d / 4) {
#pragma unroll
    for (int y = 0; y < 4; ++y) w[y] = *reinterpret_cast<const u32x4*>(vc + (int64_t)(4 * lane + y) * blk);
  }
  u32x2 kk[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = lane + 64 * u;
    if (i < n * dc) kk[u] = *reinterpret_cast<const u32x2*>(kc + 8 * i);
  }
  if (lane < d / 4) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t in[4] = {w[0][x], w[1][x], w[2][x], w[3][x]};
      uint32_t t[4];
      transpose4(in, t);
      *reinterpret_cast<u32x4*>(slab + lane * kSlabPitch + 4 * x) = u32x4{t[0], t[1], t[2], t[3]};
    }
  }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = lane + 64 * u;
    if (i >= n * dc) break;
    const int row = i / dc, cc = i - row * dc;
    const int64_t to = ((r0 + row) * c.heads + h) * d + 8 * cc;
    float f[8];
    // no page: codes of page 0 were read, and 0 is what they stand for
    const u32x2 zero = {0, 0};
    e4m3_decode8(have ? kk[u] : zero, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= ks;
    store8<DT>(ko + to, f);
    const u32x2 cd = {slab[2 * cc * kSlabPitch + row], slab[(2 * cc + 1) * kSlabPitch + row]};
    e4m3_decode8(have ? cd : zero, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= vs;
    store8<DT>(vo + to, f);
  }
}

int kv_check_cache(const cp_kv_cache* c) {
  if (!c) return set_error(CP_ERR_ARG, "null cache");
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return set_error(CP_ERR_SHAPE, "pages of %d tokens: 16, 32, 64 or 128", c->block);
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
    return set_error(CP_ERR_SHAPE, "head dimension %d: a multiple of 16 up to 256", c->head_dim);
  if (c->pages < 1 || c->pages > 0x7FFFFFFF || c->heads < 1 || c->heads > 65535)
    return set_error(CP_ERR_SHAPE, "cache of %lld pages and %d heads", (long long)c->pages, c->heads);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return set_error(CP_ERR_ARG, "null cache buffer");
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
    return set_error(CP_ERR_ALIGN, "cache codes need 16-byte and scales 4-byte alignment");
  return CP_OK;
}

int kv_check_batch(const int* table, int64_t batch, int64_t max_pages, int64_t rows, const int* offsets) {
  if (batch < 0 || max_pages < 1 || max_pages > 0x7FFFFFFF / 128 || batch > 0x7FFFFFF)
    return set_error(CP_ERR_SHAPE, "table of %lld rows of %lld pages", (long long)batch, (long long)max_pages);
  // a page of positions more than the rows still fits 32 bits
  if (rows < 0 || rows > 0x7FFFFF00) return set_error(CP_ERR_SHAPE, "%lld rows", (long long)rows);
  if (!offsets && rows != batch)
    return set_error(CP_ERR_SHAPE, "%lld rows for %lld sequences need offsets", (long long)rows, (long long)batch);
  if (batch && !table) return set_error(CP_ERR_ARG, "null table");
  return CP_OK;
}

static int kv_check_rows(const void* p, int es, int64_t row_st, int64_t head_st, const char* what) {
  if (!p) return set_error(CP_ERR_ARG, "null %s", what);
  if (!aligned(p, 16) || row_st * es % 16 || head_st * es % 16)
    return set_error(CP_ERR_ALIGN, "rows and heads of %s need 16-byte alignment", what);
  if (row_st < 0 || head_st < 0) return set_error(CP_ERR_SHAPE, "negative stride of %s", what);
  return CP_OK;
}

KvCacheArgs kv_args(const cp_kv_cache* c, const int* table, int64_t max_pages) {
  return {c->k, c->v, c->k_scale, c->v_scale, table, (int)c->pages, c->heads, c->block, c->head_dim,
          (int)max_pages};
}

}  // namespace cp

extern "C" {

int cp_kv_write(const cp_kv_cache* cache, const void* k, int64_t k_row, int64_t k_head, const void* v,
                int64_t v_row, int64_t v_head, int dtype, int64_t rows, const int32_t* table,
                int64_t batch, int64_t max_pages, const int32_t* filled, const int32_t* offsets,
                void* stream) {
  cp::clear_error();
  if (int s = cp::kv_check_cache(cache)) return s;
  if (int s = cp::kv_check_batch(table, batch, max_pages, rows, offsets)) return s;
  const int es = cp::dtype_bytes(dtype);
  if (!es) return cp::set_error(CP_ERR_ARG, "dtype code %d", dtype);
  if (rows == 0 || batch == 0) return CP_OK;
  if (!filled) return cp::set_error(CP_ERR_ARG, "null filled");
  if (int s = cp::kv_check_rows(k, es, k_row, k_head, "k")) return s;
  if (int s = cp::kv_check_rows(v, es, v_row, v_head, "v")) return s;
  // pages touched: ceil((filled % block + n) / block) summed over the sequences
  const int64_t items = offsets ? rows / cache->block + 2 * batch : batch;
  if (items * cache->heads > 4 * cp::most_workgroups(256)) return cp::set_error(CP_ERR_SHAPE, "too many rows");
  const cp::KvCacheArgs a = cp::kv_args(cache, table, max_pages);
  const cp::KvRows kr = {k, k_row, k_head}, vr = {v, v_row, v_head};
  const cp::KvBatch q = {offsets, (int)batch};
  const dim3 grid((unsigned)((items * cache->heads + 3) / 4));
  const bool keep = cache->block == 16 && cache->head_dim <= 128;
  hipStream_t st = (hipStream_t)stream;
#define CP_KV_WRITE(DT)                                                              \
  if (dtype == DT) {                                                                 \
    if (keep) cp::kv_write_kernel<DT, true><<<grid, 256, 0, st>>>(a, kr, vr, q, rows, filled); \
    else cp::kv_write_kernel<DT, false><<<grid, 256, 0, st>>>(a, kr, vr, q, rows, filled);     \
  }
  CP_KV_WRITE(CP_F32)
  CP_KV_WRITE(CP_BF16)
  CP_KV_WRITE(CP_F16)
#undef CP_KV_WRITE
  CP_LAUNCHED("cache write");
  return CP_OK;
}

int cp_kv_read(const cp_kv_cache* cache, const int32_t* table, int64_t batch, int64_t max_pages,
               const int32_t* offsets, int64_t total, void* k, void* v, int dtype, void* stream) {
  cp::clear_error();
  if (int s = cp::kv_check_cache(cache)) return s;
  if (int s = cp::kv_check_batch(table, batch, max_pages, total, offsets)) return s;
  if (!cp::dtype_bytes(dtype)) return cp::set_error(CP_ERR_ARG, "dtype code %d", dtype);
  if (total == 0) return CP_OK;
  if (!offsets) return cp::set_error(CP_ERR_ARG, "null offsets");
  if (!k || !v) return cp::set_error(CP_ERR_ARG, "null k / v");
  if (!cp::aligned(k, 16) || !cp::aligned(v, 16)) return cp::set_error(CP_ERR_ALIGN, "k and v need 16-byte alignment");
  const int64_t items = total / 16 + batch + 1;  // one more than sequences can need
  if (items * cache->heads > 4 * cp::most_workgroups(256)) return cp::set_error(CP_ERR_SHAPE, "too many rows");
  const cp::KvCacheArgs a = cp::kv_args(cache, table, max_pages);
  const cp::KvBatch q = {offsets, (int)batch};
  const dim3 grid((unsigned)((items * cache->heads + 3) / 4));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CP_F32) cp::kv_read_kernel<CP_F32><<<grid, 256, 0, st>>>(a, q, (int)items, total, (float*)k, (float*)v);
  if (dtype == CP_BF16) cp::kv_read_kernel<CP_BF16><<<grid, 256, 0, st>>>(a, q, (int)items, total, (__bf16*)k, (__bf16*)v);
  if (dtype == CP_F16) cp::kv_read_kernel<CP_F16><<<grid, 256, 0, st>>>(a, q, (int)items, total, (_Float16*)k, (_Float16*)v);
  CP_LAUNCHED("cache read");
  return CP_OK;
}

}  // extern "C"
