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

template <class T>
__device__ __forceinline__ T block_max(T v, T* lds) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) {
    const T o = __shfl_xor(v, s);
    v = v > o ? v : o;
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) v = v > lds[w] ? v : lds[w];
  __syncthreads();
  return v;
}

struct KvRows {
  const void* p;            // [rows][head][d]
  int64_t row_st, head_st;  // element strides
};

// The largest finite magnitude of n rows from row r0 of head h.
template <int DT>
__device__ __forceinline__ float kv_amax(const KvRows& x, int64_t r0, int n, int h, int d) {
  const typename Elem<DT>::T* p = (const typename Elem<DT>::T*)x.p + r0 * x.row_st + h * x.head_st;
  float m = 0.0f;
  const int dc = d / 8;
  for (int c = threadIdx.x; c < n * dc; c += 256) {
    const int row = c / dc;
    float v[8];
    load8<DT>(p + row * x.row_st + 8 * (c - row * dc), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(v[i]);
      m = a < __builtin_inff() && a > m ? a : m;
    }
  }
  return m;
}

// Eight scaled values' codes.
template <int DT>
__device__ __forceinline__ u32x2 kv_codes(const typename Elem<DT>::T* p, float inv) {
  float v[8];
  load8<DT>(p, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = kv_clamp(v[i] * inv);
  return e4m3_encode8(v);
}

__device__ __forceinline__ uint8_t kv_rescale(uint8_t c, float ratio) {
  const float v = __builtin_amdgcn_cvt_f32_fp8((int)c, 0) * ratio;
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false);
}

// One workgroup per (touched page, head). It takes the page's scales from the rows that
// fall into it, moves the codes held to a larger scale where it has to, and writes the
// rows' codes: K as they come, V through LDS, transposed. Bound by HBM for prompts, by
// latency for single tokens.
template <int DT>
__global__ __launch_bounds__(256) void kv_write_kernel(KvCacheArgs c, KvRows k, KvRows v,
                                                       KvBatch q, int64_t rows, const int* filled) {
  extern __shared__ __align__(16) uint8_t tile[];  // [n][d + 4]: V codes by token
  __shared__ float red[4];
  const int h = (int)(blockIdx.x % c.heads);
  int b, item, n_b;
  int64_t row0;
  const bool ok = kv_locate(
      q, (int)(blockIdx.x / c.heads),
      [&](int s, int n) { return n ? (max(filled[s], 0) % c.block + n + c.block - 1) / c.block : 0; },
      &b, &item, &row0, &n_b);
  if (!ok) return;
  const int held = max(filled[b], 0);
  const int64_t pg = (int64_t)held / c.block + item;  // page of the sequence
  const int s0 = item == 0 ? held % c.block : 0;      // first slot written
  const int done = item == 0 ? 0 : item * c.block - held % c.block;  // rows in earlier pages
  const int n = min(n_b - done, c.block - s0);
  const int64_t r0 = row0 + done;
  if (pg >= c.max_pages || r0 < 0 || r0 + n > rows) return;
  const int page = c.table[(int64_t)b * c.max_pages + pg];
  if ((unsigned)page >= (unsigned)c.pages) return;
  const int64_t ph = (int64_t)page * c.heads + h;
  const int d = c.d, blk = c.block, dc = d / 8;
  uint8_t* kc = c.k + ph * blk * d;
  uint8_t* vc = c.v + ph * blk * d;

  const float ka = block_max(kv_amax<DT>(k, r0, n, h, d), red);
  const float va = block_max(kv_amax<DT>(v, r0, n, h, d), red);
  float ks = kv_scale(ka), vs = kv_scale(va);
  if (s0 > 0) {  // codes held: keep the larger scale
    const float ko = c.k_scale[ph], vo = c.v_scale[ph];
    if (ks > ko) {
      const float ratio = ko * inv_pow2(ks);
      for (int i = threadIdx.x; i < s0 * d; i += 256) kc[i] = kv_rescale(kc[i], ratio);
    } else {
      ks = ko;
    }
    if (vs > vo) {
      const float ratio = vo * inv_pow2(vs);
      for (int i = threadIdx.x; i < s0 * d; i += 256) {
        const int at = i / s0 * blk + i % s0;
        vc[at] = kv_rescale(vc[at], ratio);
      }
    } else {
      vs = vo;
    }
  }
  __syncthreads();  // every thread has read the old scales
  if (threadIdx.x == 0) {
    c.k_scale[ph] = ks;
    c.v_scale[ph] = vs;
  }
  typedef typename Elem<DT>::T T;
  const T* kp = (const T*)k.p + r0 * k.row_st + h * k.head_st;
  const T* vp = (const T*)v.p + r0 * v.row_st + h * v.head_st;
  const float ki = inv_pow2(ks), vi = inv_pow2(vs);
  const int pitch = d + 4;
  for (int i = threadIdx.x; i < n * dc; i += 256) {
    const int row = i / dc, col = 8 * (i - row * dc);
    *reinterpret_cast<u32x2*>(kc + (int64_t)(s0 + row) * d + col) = kv_codes<DT>(kp + row * k.row_st + col, ki);
    const u32x2 cv = kv_codes<DT>(vp + row * v.row_st + col, vi);
    *reinterpret_cast<uint32_t*>(tile + row * pitch + col) = cv[0];
    *reinterpret_cast<uint32_t*>(tile + row * pitch + col + 4) = cv[1];
  }
  __syncthreads();
  const int groups = blk / 16;
  for (int i = threadIdx.x; i < d * groups; i += 256) {
    const int col = i % d, g = i / d;
    const int lo = max(s0, 16 * g), hi = min(s0 + n, 16 * g + 16);
    if (lo >= hi) continue;
    uint8_t* out = vc + (int64_t)col * blk + 16 * g;
    if (hi - lo == 16) {
      u32x4 w = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j / 4] |= (uint32_t)tile[(16 * g + j - s0) * pitch + col] << (8 * (j % 4));
      *reinterpret_cast<u32x4*>(out) = w;
    } else {
      for (int j = lo; j < hi; ++j) out[j - 16 * g] = tile[(j - s0) * pitch + col];
    }
  }
}

// One workgroup per (page held, head): the codes' values in rows [total][head][d].
template <int DT>
__global__ __launch_bounds__(256) void kv_read_kernel(KvCacheArgs c, KvBatch q, int64_t total,
                                                      typename Elem<DT>::T* __restrict__ ko,
                                                      typename Elem<DT>::T* __restrict__ vo) {
  extern __shared__ __align__(16) uint8_t tile[];  // [block][d + 4]
  const int h = (int)(blockIdx.x % c.heads);
  int b, item, n_b;
  int64_t row0;
  if (!kv_locate(q, (int)(blockIdx.x / c.heads),
                 [&](int, int n) { return (n + c.block - 1) / c.block; }, &b, &item, &row0, &n_b))
    return;
  const int n = min(n_b - item * c.block, c.block);
  const int64_t r0 = row0 + (int64_t)item * c.block;
  if (r0 < 0 || r0 + n > total) return;
  const int page = item < c.max_pages ? c.table[(int64_t)b * c.max_pages + item] : -1;
  const bool have = (unsigned)page < (unsigned)c.pages;
  const int64_t ph = have ? (int64_t)page * c.heads + h : 0;
  const int d = c.d, blk = c.block, dc = d / 8, pitch = d + 4;
  const uint8_t* kc = c.k + ph * blk * d;
  const uint8_t* vc = c.v + ph * blk * d;
  const float ks = have ? c.k_scale[ph] : 0.0f, vs = have ? c.v_scale[ph] : 0.0f;
  for (int i = threadIdx.x; i < d * (blk / 16); i += 256) {
    const int col = i % d, g = i / d;
    if (16 * g >= n) continue;
    u32x4 w = {0, 0, 0, 0};
    if (have) w = *reinterpret_cast<const u32x4*>(vc + (int64_t)col * blk + 16 * g);
#pragma unroll
    for (int j = 0; j < 16; ++j) tile[(16 * g + j) * pitch + col] = (uint8_t)(w[j / 4] >> (8 * (j % 4)));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * dc; i += 256) {
    const int row = i / dc, col = 8 * (i - row * dc);
    const int64_t at = ((r0 + row) * c.heads + h) * d + col;
    u32x2 cd = {0, 0};
    if (have) cd = *reinterpret_cast<const u32x2*>(kc + (int64_t)row * d + col);
    float f[8];
    e4m3_decode8(cd, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= ks;
    store8<DT>(ko + at, f);
    cd[0] = *reinterpret_cast<const uint32_t*>(tile + row * pitch + col);
    cd[1] = *reinterpret_cast<const uint32_t*>(tile + row * pitch + col + 4);
    e4m3_decode8(cd, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= vs;
    store8<DT>(vo + at, f);
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
  if (rows < 0 || rows > 0x7FFFFFFF) return set_error(CP_ERR_SHAPE, "%lld rows", (long long)rows);
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
  if (items * cache->heads > 0x7FFFFFFF) return cp::set_error(CP_ERR_SHAPE, "too many rows");
  const cp::KvCacheArgs a = cp::kv_args(cache, table, max_pages);
  const cp::KvRows kr = {k, k_row, k_head}, vr = {v, v_row, v_head};
  const cp::KvBatch q = {offsets, (int)batch};
  const dim3 grid((unsigned)(items * cache->heads));
  const size_t lds = (size_t)cache->block * (cache->head_dim + 4);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CP_F32) cp::kv_write_kernel<CP_F32><<<grid, 256, lds, st>>>(a, kr, vr, q, rows, filled);
  if (dtype == CP_BF16) cp::kv_write_kernel<CP_BF16><<<grid, 256, lds, st>>>(a, kr, vr, q, rows, filled);
  if (dtype == CP_F16) cp::kv_write_kernel<CP_F16><<<grid, 256, lds, st>>>(a, kr, vr, q, rows, filled);
  CP_LAUNCHED("cache write");
  return CP_OK;
}

int cp_kv_read(const cp_kv_cache* cache, const int32_t* table, int64_t batch, int64_t max_pages,
               const int32_t* offsets, int64_t total, void* k, void* v, int dtype, void* stream) {
  cp::clear_error();
  if (int s = cp::kv_check_cache(cache)) return s;
  if (int s = cp::kv_check_batch(table, batch, max_pages, total, offsets)) return s;
  if (!cp::dtype_bytes(dtype)) return cp::set_error(CP_ERR_ARG, "dtype code %d", dtype);
  if (total == 0 || batch == 0) return CP_OK;
  if (!offsets) return cp::set_error(CP_ERR_ARG, "null offsets");
  if (!k || !v) return cp::set_error(CP_ERR_ARG, "null k / v");
  if (!cp::aligned(k, 16) || !cp::aligned(v, 16)) return cp::set_error(CP_ERR_ALIGN, "k and v need 16-byte alignment");
  const int64_t items = total / cache->block + batch;
  if (items * cache->heads > 0x7FFFFFFF) return cp::set_error(CP_ERR_SHAPE, "too many rows");
  const cp::KvCacheArgs a = cp::kv_args(cache, table, max_pages);
  const cp::KvBatch q = {offsets, (int)batch};
  const dim3 grid((unsigned)(items * cache->heads));
  const size_t lds = (size_t)cache->block * (cache->head_dim + 4);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CP_F32) cp::kv_read_kernel<CP_F32><<<grid, 256, lds, st>>>(a, q, total, (float*)k, (float*)v);
  if (dtype == CP_BF16) cp::kv_read_kernel<CP_BF16><<<grid, 256, lds, st>>>(a, q, total, (__bf16*)k, (__bf16*)v);
  if (dtype == CP_F16) cp::kv_read_kernel<CP_F16><<<grid, 256, lds, st>>>(a, q, total, (_Float16*)k, (_Float16*)v);
  CP_LAUNCHED("cache read");
  return CP_OK;
}

}  // extern "C"
