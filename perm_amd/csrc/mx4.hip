// MXFP4 (microscaled 4-bit floating point) on gfx950: quantisation, decode and product.
//
// A block is 32 consecutive values of a row with one power-of-two scale 2^e. With
// a = max |x| over the block,
//     e = floor(log2 a) - 2 (at least -127),  code = RNE to e2m1 of x * 2^-e,  |code| <= 6
// so the largest magnitude lands in [4, 8) and saturates at 6. A block with a NaN or an
// infinity gets the scale byte 255 and decodes to NaN; an all-zero block gets byte 0.
// Scaling by a power of two is exact, so the e2m1 rounding is the only one.
//
// Layout. codes [rows][k / 2], two a byte, the even column in the low four bits. The scale
// bytes (e + 127) lie as v_mfma_scale_f32_16x16x128_f8f6f4 takes them: its lane l holds row
// l % 16 and the 32-block l / 16 of a 128-wide step, and picks one byte of a dword by an
// immediate. So the dword of (step s, row group R of 64, lane l) holds that lane's four
// 16-row tiles: byte ((s * ceil(rows / 64) + R) * 64 + l) * 4 + j is the scale of row
// 64 R + 16 j + l % 16, block 4 s + l / 16. One 256-byte load serves 64 rows of a step.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "lowbit.h"

namespace cp {

// f(integral_constant 0), f(1), ... f(N - 1): indices that builtins take as immediates.
template <class F, int... I>
__device__ __forceinline__ void unrolled_impl(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled_impl(f, std::make_integer_sequence<int, N>{});
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kMxBlock = 32;    // values that share a scale
constexpr int kMxStep = 128;    // values of one MFMA step
constexpr int kMxGroup = 64;    // rows that share a scale dword's bytes

inline int64_t mx_steps(int64_t k) { return (k + kMxStep - 1) / kMxStep; }
inline int64_t mx_groups(int64_t rows) { return (rows + kMxGroup - 1) / kMxGroup; }

// The scale byte of a block whose largest magnitude is a (NaN or infinity: 255).
__device__ __forceinline__ int mx_scale_byte(float a) {
  if (!(a < __builtin_inff())) return 255;
  const int e = a == 0.0f ? -127 : frexp_e(a) - 3;
  return (e < -127 ? -127 : e) + 127;
}

// 2^-e of a scale byte; e <= 125, so it is never below 2^-125.
__device__ __forceinline__ float mx_inv_scale(int byte) {
  return __uint_as_float((uint32_t)(254 - byte) << 23);
}

// Eight values' codes packed in a dword (values already scaled; saturating at 6).
__device__ __forceinline__ uint32_t mx_pack8(const float (&v)[8], float inv) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0] * inv, v[1] * inv, 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2] * inv, v[3] * inv, 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4] * inv, v[5] * inv, 1.0f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6] * inv, v[7] * inv, 1.0f, 3);
  return c;
}

// max |v| over the four lanes that hold a block, NaN if any value is one.
__device__ __forceinline__ float mx_block_amax(const float (&v)[8]) {
  uint32_t m = 0;
  // |v| compares as an integer: infinity and NaN sort above every finite magnitude
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
    m = m > b ? m : b;
  }
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true);
  m = m > o ? m : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true);
  return __uint_as_float(m > o ? m : o);
}

// One workgroup per (128 columns, 64 rows): thread t takes columns 8 (t % 16) .. + 7 of the
// rows t / 16 + 16 j, j = 0..3, so four lanes share a block and the four bytes of a scale
// dword come from one thread. Bound by HBM: each value is read once, each byte written once
// (14336 x 4096 in float32 with the decode after it: 532 MB in 106.6 us, 104 at a copy's 5.1
// TB/s). A token's row is a launch of 2.7 us.
template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const typename Elem<DT>::T* __restrict__ x,
                                                           int64_t rows, int k, int64_t stride,
                                                           uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales) {
  const int t = threadIdx.x, step = blockIdx.x;
  const int64_t group = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  const int64_t groups = (rows + kMxGroup - 1) / kMxGroup;
  if (group >= groups) return;
  const int col = step * kMxStep + 8 * (t & 15);
  float v[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = group * kMxGroup + 16 * j + (t >> 4);
    if (r < rows && col < k) {
      load8<DT>(x + r * stride + col, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
    }
  }
  uint32_t bytes = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = group * kMxGroup + 16 * j + (t >> 4);
    const int b = mx_scale_byte(mx_block_amax(v[j]));
    bytes |= (uint32_t)b << (8 * j);
    if (r < rows && col < k)
      *reinterpret_cast<uint32_t*>(codes + r * (k / 2) + col / 2) =
          b == 255 ? 0u : mx_pack8(v[j], mx_inv_scale(b));
  }
  if ((t & 3) == 0)
    *reinterpret_cast<uint32_t*>(
        scales + ((step * groups + group) * 64 + 16 * ((t & 15) >> 2) + (t >> 4)) * 4) = bytes;
}

// The values of eight codes: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6.
__device__ __forceinline__ void mx_unpack8(uint32_t c, float scale, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
  const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[i] = a[i] * scale;
    v[2 + i] = b[i] * scale;
    v[4 + i] = d[i] * scale;
    v[6 + i] = e[i] * scale;
  }
}

// The decode, over the same tiles as the quantiser and bound as it is.
template <int DT>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales,
                                                             int64_t rows, int k,
                                                             typename Elem<DT>::T* __restrict__ y) {
  const int t = threadIdx.x, step = blockIdx.x;
  const int64_t group = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  const int64_t groups = (rows + kMxGroup - 1) / kMxGroup;
  if (group >= groups) return;
  const int col = step * kMxStep + 8 * (t & 15);
  if (col >= k) return;
  const uint32_t bytes = *reinterpret_cast<const uint32_t*>(
      scales + ((step * groups + group) * 64 + 16 * ((t & 15) >> 2) + (t >> 4)) * 4);
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = group * kMxGroup + 16 * j + (t >> 4);
    c[j] = r < rows ? *reinterpret_cast<const uint32_t*>(codes + r * (k / 2) + col / 2) : 0;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = group * kMxGroup + 16 * j + (t >> 4);
    if (r >= rows) break;
    float v[8];
    mx_unpack8(c[j], pow2_byte((bytes >> (8 * j)) & 255), v);
    store8<DT>(y + r * k + col, v);
  }
}

// ---------------------------------------------------------------- product
// Y[m][n] = sum over k of a[m][k] b[n][k]. b's rows are the MFMA's A operand, so a lane's
// four results are consecutive n of one m.

struct MxOperand {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows;
};

// c += a b over one step; SA and SB: which byte of the scale dwords is the operand's.
template <int SA, int SB>
__device__ __forceinline__ f32x4 mx_mfma(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, SA, (int)sa, SB, (int)sb);
}

template <int DT>
__device__ __forceinline__ void mx_store4(typename Elem<DT>::T* y, int64_t m, int64_t n0, int64_t M,
                                          int64_t N, f32x4 c) {
  if (m >= M) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < N) y[m * N + n0 + i] = (typename Elem<DT>::T)c[i];
}

// Few rows of a (at most 32): bound by reading b once (1 x 14336 x 4096: 31 MB in 6.2 us, 5.0
// TB/s, most of it from the last-level cache), and by a launch's own 3 us where b is small. A
// workgroup takes NT 16-row tiles of b and all of a; its waves take the 128-column steps in
// turn, four or eight steps' loads in flight in each, and join their sums in LDS in wave order.
// b's codes go from memory to the matrix cores without LDS: each is used once. Four
// neighbouring workgroups of one XCD share the scale dwords of 64 rows in its L2.
//
// XT >= 0: a's rows come as values of that type and are quantized by every workgroup into
// its LDS ([row][k / 2] codes, then [row][k / 32] scale bytes), beside the first loads of b.
constexpr int kFewWaves = 4;

template <int MT, int NT, int XT, int DT>
__global__ __launch_bounds__(XT >= 0 ? 1024 : 64 * kFewWaves) void mx4_few_kernel(
    MxOperand a, MxOperand b, const void* x, int64_t stride, int k, int wgs, typename Elem<DT>::T* __restrict__ y) {
  constexpr int U = MT + NT > 2 ? 4 : 8;
  constexpr bool FUSED = XT >= 0;
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, g = lane >> 4, W = FUSED ? blockDim.x >> 6 : kFewWaves;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // blocks of 32 workgroups: XCD x (w % 8) takes four neighbours
  int w = blockIdx.x;
  if ((w | 31) < wgs) w = (w & ~31) + 4 * (w & 7) + ((w & 31) >> 3);
  const int64_t n0 = (int64_t)w * NT * 16;
  const int steps = (k + kMxStep - 1) / kMxStep, M = (int)a.rows, kb = k / 2, nblk = k / kMxBlock;
  const int64_t ga = (a.rows + 63) / 64, gb = (b.rows + 63) / 64;
  const uint32_t* sb = reinterpret_cast<const uint32_t*>(b.scales) + (n0 / 64) * 64 + lane;
  const uint32_t* sa = reinterpret_cast<const uint32_t*>(a.scales) + lane;
  const int jb = (int)(n0 / 16 & 3) * 8;
  const uint8_t* pb[NT];
  const uint8_t* pa[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) pb[j] = b.codes + min(n0 + 16 * j + (lane & 15), b.rows - 1) * kb + 16 * g;
#pragma unroll
  for (int i = 0; i < MT; ++i) pa[i] = a.codes + min((int64_t)(16 * i + (lane & 15)), a.rows - 1) * kb + 16 * g;

  u32x4 fb[U][NT], fa[U][MT];
  uint32_t vb[U], va[U];
  const u32x4 zero = {0, 0, 0, 0};
  // step s = base + W u + wave: rows past the end repeat the last (never stored), columns
  // past the end are zero codes in a
  auto load_b = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = base + W * u + wave, blk = 4 * s + g;
      vb[u] = sb[min(s, steps - 1) * gb * 64] >> jb;
#pragma unroll
      for (int j = 0; j < NT; ++j)
        fb[u][j] = blk < nblk ? *reinterpret_cast<const u32x4*>(pb[j] + (int64_t)s * 64) : zero;
    }
  };
  const int pitch = kb + 16;
  auto load_a = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = base + W * u + wave, blk = 4 * s + g;
      if constexpr (FUSED) {
        va[u] = 0;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int m = 16 * i + (lane & 15);
          const bool in = blk < nblk && m < M;
          fa[u][i] = in ? *reinterpret_cast<const u32x4*>(lds + m * pitch + 16 * blk) : zero;
          va[u] |= in ? (uint32_t)lds[M * pitch + m * nblk + blk] << (8 * i) : 0;
        }
      } else {
        va[u] = sa[min(s, steps - 1) * ga * 64];
#pragma unroll
        for (int i = 0; i < MT; ++i)
          fa[u][i] = blk < nblk ? *reinterpret_cast<const u32x4*>(pa[i] + (int64_t)s * 64) : zero;
      }
    }
  };
  load_b(0);
  if constexpr (FUSED) {
    typedef typename Elem<XT>::T T;
    const int chunks = k / 8;  // k % 32 == 0: four lanes hold a block
#pragma unroll 4
    for (int t = threadIdx.x; t < M * chunks; t += 64 * W) {
      const int m = t / chunks, c = t - m * chunks;
      float v[8];
      load8<XT>((const T*)x + m * stride + 8 * c, v);
      const int e = mx_scale_byte(mx_block_amax(v));
      *reinterpret_cast<uint32_t*>(lds + m * pitch + 4 * c) = e == 255 ? 0u : mx_pack8(v, mx_inv_scale(e));
      if ((c & 3) == 0) lds[M * pitch + m * nblk + (c >> 2)] = (uint8_t)e;
    }
    __syncthreads();
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  load_a(0);
  for (int base = 0;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unrolled<MT>([&](auto I) {
        unrolled<NT>([&](auto J) {
          acc[I][J] = mx_mfma<J, I>(fb[u][J], fa[u][I], acc[I][J], vb[u], va[u]);
        });
      });
    }
    base += U * W;
    if (base >= steps) break;
    load_b(base);
    load_a(base);
  }
  // the waves' sums, joined in wave order; a slot is one lane's four results
  f32x4* red = reinterpret_cast<f32x4*>(lds);
  if constexpr (FUSED) __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[(wave * MT * NT + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int t = threadIdx.x; t < MT * NT * 64; t += 64 * W) {
    f32x4 c = red[t];
    for (int v = 1; v < W; ++v) c += red[v * MT * NT * 64 + t];
    const int l = t & 63, ij = t >> 6;
    const int64_t m = 16 * (ij / NT) + (l & 15), n = n0 + 16 * (ij % NT) + 4 * (l >> 4);
    if (DT != CP_F32 && (b.rows & 3) == 0) {
      if (m < M && n < b.rows) {
        u32x2 p;
        p[0] = pack2<DT>(c[0], c[1]);
        p[1] = pack2<DT>(c[2], c[3]);
        *reinterpret_cast<u32x2*>(y + m * b.rows + n) = p;
      }
    } else {
      mx_store4<DT>(y, m, n, a.rows, b.rows, c);
    }
  }
}

// A wave's FM x FN tiles of results to y. 16-bit results whose rows are 16-byte aligned go
// through the wave's own LDS region, [16 FM][16 FN] with 16-byte chunks permuted by xor with
// the row, and leave in whole row segments; others go straight from the registers.
template <int FM, int FN, int DT>
__device__ __forceinline__ void mx_store_tile(typename Elem<DT>::T* y, int64_t m0, int64_t n0, int64_t M,
                                              int64_t N, const f32x4 (&acc)[FM][FN], uint8_t* lds) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  if (DT != CP_F32 && (N & 7) == 0) {
    constexpr int CH = 2 * FN, MASK = (CH < 16 ? CH : 16) - 1;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r = 16 * i + (lane & 15);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        u32x2 w;
        w[0] = pack2<DT>(acc[i][j][0], acc[i][j][1]);
        w[1] = pack2<DT>(acc[i][j][2], acc[i][j][3]);
        const int c = (2 * j + (g >> 1)) ^ (r & MASK);
        *reinterpret_cast<u32x2*>(lds + (r * CH + c) * 16 + 8 * (g & 1)) = w;
      }
    }
    constexpr int RPI = 64 / CH;  // rows a store covers
#pragma unroll
    for (int i = 0; i < 16 * FM / RPI; ++i) {
      const int r = i * RPI + lane / CH, c = lane % CH;
      const u32x4 w = *reinterpret_cast<const u32x4*>(lds + (r * CH + (c ^ (r & MASK))) * 16);
      const int64_t m = m0 + r, n = n0 + 8 * c;
      if (m < M && n < N) *reinterpret_cast<u32x4*>(y + m * N + n) = w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t m = m0 + 16 * i + (lane & 15);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t n = n0 + 16 * j + 4 * g;
      if (DT == CP_F32 && (N & 3) == 0) {
        if (m < M && n < N) *reinterpret_cast<f32x4*>(y + m * N + n) = acc[i][j];
      } else {
        mx_store4<DT>(y, m, n, M, N, acc[i][j]);
      }
    }
  }
}

// Large products, bound by the matrix cores where the tiles fill the GPU (8192 x 8192 x 8192 of
// normal values: 228 to 238 us, 4.6 to 4.8 PFLOP/s; the instruction alone reaches 5.9 on random
// codes, where power limits it) and by a tile's start and end where there are few stages
// (4096 x 14336 x 4096: 3.5 rounds of tiles, 117 us, 4.1 PFLOP/s; of uniformly random codes, which
// draw more power, 124 to 142). A workgroup of WM x WN waves owns a tile of BM x BN results, each wave
// FM x FN MFMA tiles of it. 256 columns of both operands are staged in LDS a step ahead by
// loads that write LDS directly, 16 bytes a lane, in two buffers; a row's eight 16-byte
// chunks are permuted by xor with the row's low three bits, so that the 16 rows of an operand
// read spread over the banks. The direct loads fill LDS in lane order, so the permutation is
// applied to the address they read. Scales come straight from memory, one dword a lane for
// 64 rows and 128 columns.
constexpr int kStage = 256;               // columns per stage
constexpr int kStageBytes = kStage / 2;   // bytes per row
constexpr uint32_t kOob = 0x80000000u;    // past any tile's bytes (at most 256 * 2^22)

typedef __attribute__((address_space(3))) void* lptr_t;

template <int WM, int WN, int FM, int FN, int DT>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx4_gemm_kernel(MxOperand a, MxOperand b, int k, int mt, int nt,
                                                                   int splits, typename Elem<DT>::T* __restrict__ y) {
  constexpr int W = WM * WN, BM = 16 * WM * FM, BN = 16 * WN * FN, ROWS = BM + BN;
  constexpr int LA = BM / (8 * W), LB = BN / (8 * W);  // direct loads of a wave per stage, 8 rows each
  constexpr int DA = FM > 4 ? FM / 4 : 1, DB = FN > 4 ? FN / 4 : 1;
  static_assert(LA * 8 * W == BM && LB * 8 * W == BN && FM % 2 == 0, "tile shape");
  extern __shared__ __align__(16) uint8_t lds[];  // [2][ROWS][128]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // Workgroup w runs on XCD w % 8. Each XCD takes a contiguous run of tiles, ordered in
  // columns of eight m tiles, so that the tiles in flight on one XCD form a block and share
  // their operands in its L2.
  int tm, tn, split;
  {
    const int tiles = mt * nt * splits, w = blockIdx.x;
    const int x = w & 7, q = tiles >> 3, r = tiles & 7;
    int t = x * q + min(x, r) + (w >> 3);
    split = t / (mt * nt);
    t -= split * mt * nt;
    const int col = t / (8 * nt), h = min(8, mt - 8 * col), u = t - col * 8 * nt;
    tn = u / h;
    tm = 8 * col + u % h;
  }
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int kb = k / 2, blocks = k / kMxBlock;
  // columns in stages of 256; a split takes an equal run of them and its own [rows][rows] sums
  const int stages = (k + kStage - 1) / kStage, steps = (k + kMxStep - 1) / kMxStep;
  const int sb0 = split * stages / splits, sb1 = (split + 1) * stages / splits;
  y += split * a.rows * b.rows;

  // Buffer loads over the tile's rows: a row past the operand's end, and a lane whose chunk
  // lies past the end of a row (given an offset past any buffer), reads zeros. A zero code
  // adds nothing. Wave w loads rows 8 (LA w + i) + lane / 8 of a and the like of b.
  const int chunk = (lane & 7) ^ (lane >> 3);
  const auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)(a.codes + m0 * kb), 0,
                                                    (int)(min((int64_t)BM, a.rows - m0) * kb), 0x00020000);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)(b.codes + n0 * kb), 0,
                                                    (int)(min((int64_t)BN, b.rows - n0) * kb), 0x00020000);
  const uint32_t va = (uint32_t)(8 * LA * wave + (lane >> 3)) * kb + 16 * chunk;
  const uint32_t vb = (uint32_t)(8 * LB * wave + (lane >> 3)) * kb + 16 * chunk;
  constexpr int L = LA + LB;
  auto fetch = [&](int s, int i0, int i1) {  // loads i0 .. i1 - 1 of stage s
    uint8_t* to = lds + (s & 1) * ROWS * kStageBytes;
    const bool in = chunk < blocks - 8 * s;
    const int at = __builtin_amdgcn_readfirstlane(s * kStageBytes);
#pragma unroll
    for (int i = i0; i < i1; ++i) {
      if (i < LA)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lptr_t)(to + (LA * wave + i) * 1024), 16,
                                                 in ? va + 8 * i * kb : kOob, at, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lptr_t)(to + BM * kStageBytes + (LB * wave + i - LA) * 1024), 16,
                                                 in ? vb + 8 * (i - LA) * kb : kOob, at, 0, 0);
    }
  };
  const int64_t ga = (a.rows + 63) / 64, gb = (b.rows + 63) / 64;
  uint32_t sa[2][DA], sb[2][DB], na[2][DA], nb[2][DB];  // [step][64-row group], this stage and next
  const uint32_t* pa[DA];
  const uint32_t* pb[DB];
#pragma unroll
  for (int i = 0; i < DA; ++i)
    pa[i] = reinterpret_cast<const uint32_t*>(a.scales) + min(m0 / 64 + wm * FM / 4 + i, ga - 1) * 64 + lane;
#pragma unroll
  for (int i = 0; i < DB; ++i)
    pb[i] = reinterpret_cast<const uint32_t*>(b.scales) + min(n0 / 64 + wn * FN / 4 + i, gb - 1) * 64 + lane;
  auto fetch_scales = [&](int s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t st = min(2 * s + j, steps - 1);
#pragma unroll
      for (int i = 0; i < DA; ++i) na[j][i] = pa[i][st * ga * 64] >> (FM < 4 ? 8 * (wm * FM & 3) : 0);
#pragma unroll
      for (int i = 0; i < DB; ++i) nb[j][i] = pb[i][st * gb * 64] >> (FN < 4 ? 8 * (wn * FN & 3) : 0);
    }
  };
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // operand reads: row lane % 16, chunk 4 step + lane / 16, permuted by the row's low bits
  const int row = lane & 15;
  const int at0 = row * kStageBytes + 16 * ((lane >> 4) ^ (row & 7));
  const int at1 = row * kStageBytes + 16 * ((4 + (lane >> 4)) ^ (row & 7));
  u32x4 fa[FM], fb[2][FN];  // fb by step of the stage
  auto read_a = [&](int s, auto P, int i) {
    fa[i] = *reinterpret_cast<const u32x4*>(lds + (s & 1) * ROWS * kStageBytes + (wm * FM + i) * 16 * kStageBytes +
                                            (P ? at1 : at0));
  };
  auto read_b = [&](int s, auto P, int j) {
    fb[P][j] = *reinterpret_cast<const u32x4*>(lds + (s & 1) * ROWS * kStageBytes +
                                               (BM + (wn * FN + j) * 16) * kStageBytes + (P ? at1 : at0));
  };
  auto mfmas = [&](auto P, auto I) {
    unrolled<FN>([&](auto J) {
      acc[I][J] = mx_mfma<J % 4, I % 4>(fb[P][J], fa[I], acc[I][J], sb[P][J / 4], sa[P][I / 4]);
    });
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> P0{};
  constexpr std::integral_constant<int, 1> P1{};
  // The pipeline. Each row of FN MFMAs is issued with the operand reads of later rows, so
  // no MFMA waits for a read issued just before it. A stage's last reads are issued halfway
  // through its second step; there the workgroup meets once, the next stage has landed (it
  // was fetched a stage ago), the buffer just read is free for the stage after it, and the
  // rest of the step's MFMAs cover the first reads of the next stage. The fetches are spread
  // over rows of MFMAs: a wave that issues eight at once waits for the address unit, which
  // takes 16 clocks for each, while its MFMAs behind them wait too.
  auto scales_now = [&] {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < DA; ++i) sa[j][i] = na[j][i];
#pragma unroll
      for (int i = 0; i < DB; ++i) sb[j][i] = nb[j][i];
    }
  };
  constexpr int HM = FM / 2, AHEAD = FM > 2 ? 2 : 1;  // a row read ahead must not be one still in use
  fetch(sb0, 0, L);
  fetch_scales(sb0);
  __syncthreads();
  fetch(sb0 + 1, 0, L / 2);
  scales_now();
#pragma unroll
  for (int j = 0; j < FN; ++j) read_b(sb0, P0, j);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) read_a(sb0, P0, i);
#pragma clang loop unroll(disable)
  for (int s = sb0; s < sb1; ++s) {
    unrolled<FM>([&](auto I) {
      if constexpr (I < HM) fetch(s + 1, L / 2 + I * L / FM, L / 2 + (I + 1) * L / FM);
      if constexpr (I == HM) fetch_scales(s + 1);
      if constexpr (I + AHEAD < FM) read_a(s, P0, I + AHEAD);
      else read_a(s, P1, I + AHEAD - FM);
#pragma unroll
      for (int j = I * FN / FM; j < (I + 1) * FN / FM; ++j) read_b(s, P1, j);
      mfmas(P0, I);
    });
    unrolled<HM>([&](auto I) {
#pragma unroll
      for (int i = AHEAD + I * (FM - AHEAD) / HM; i < AHEAD + (I + 1) * (FM - AHEAD) / HM; ++i) read_a(s, P1, i);
      mfmas(P1, I);
    });
    __syncthreads();
    unrolled<FM - HM>([&](auto I) {
      fetch(s + 2, I * L / FM, (I + 1) * L / FM);
#pragma unroll
      for (int j = I * FN / (FM - HM); j < (I + 1) * FN / (FM - HM); ++j) read_b(s + 1, P0, j);
      if constexpr (I < AHEAD) read_a(s + 1, P0, I);
      mfmas(P1, std::integral_constant<int, I + HM>{});
    });
    scales_now();
  }
  __syncthreads();  // the last fetches (zeros) are in before LDS is used again or given up
  mx_store_tile<FM, FN, DT>(y, m0 + wm * FM * 16, n0 + wn * FN * 16, a.rows, b.rows, acc,
                            lds + wave * FM * FN * 512);
}

// y = the splits' sums in split order. Bound by reading them: 4 bytes a split and result.
template <int DT>
__global__ __launch_bounds__(256) void mx4_join_kernel(const float* __restrict__ part, int64_t count, int splits,
                                                       typename Elem<DT>::T* __restrict__ y) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i + 4 <= count && (count & 3) == 0) {
    f32x4 c = *reinterpret_cast<const f32x4*>(part + i);
    for (int s = 1; s < splits; ++s) c += *reinterpret_cast<const f32x4*>(part + s * count + i);
    if constexpr (DT == CP_F32) {
      *reinterpret_cast<f32x4*>(y + i) = c;
    } else {
      u32x2 p;
      p[0] = pack2<DT>(c[0], c[1]);
      p[1] = pack2<DT>(c[2], c[3]);
      *reinterpret_cast<u32x2*>(y + i) = p;
    }
  } else {
    for (int64_t j = i; j < i + 4 && j < count; ++j) {
      float c = part[j];
      for (int s = 1; s < splits; ++s) c += part[s * count + j];
      y[j] = (typename Elem<DT>::T)c;
    }
  }
}

// How a product of m x n results over k columns is cut up.
struct MxPlan {
  int few;     // a's rows in tiles of 16 on mx4_few_kernel, or 0
  int edge;    // otherwise the edge of mx4_gemm_kernel's square tiles: 64, 128 or 256
  int splits;  // of the columns
};

// Tiles are chosen by predicted time. A stage takes a tile of edge 64 / 128 / 256 at least
// 0.47 / 0.73 / 1.9 us however empty the GPU is, and a CU with several tiles 0.23 / 0.69 /
// 1.9 us a tile (measured at k = 4096: 512 x 4096 results 11.6 / 13.2 / 23.5 us, 256 x 14336
// 18.4 / 15.2 / 25.1, 1024 x 14336 52 / 38 / 33). Columns are split while that leaves at least
// 12 stages a split and no more than two small tiles (or one) a CU, where joining costs less
// than it saves (over 14336 columns 128 x 4096 results take 17.5 us in four splits, 26.6 in
// one; 1024 x 4096, in 256 tiles of 128, 44.7 in two and 41.1 in one).
static MxPlan mx_plan(int64_t m, int64_t n, int64_t k) {
  if (m <= 32) return {(int)((m + 15) / 16), 0, 1};
  const int edges[3] = {64, 128, 256};
  const double least[3] = {0.47, 0.73, 1.9}, each[3] = {0.23, 0.69, 1.9};
  MxPlan p = {0, 0, 1};
  double best = 0.0;
  int64_t tiles = 1;
  for (int i = 0; i < 3; ++i) {
    const int64_t t = ((m + edges[i] - 1) / edges[i]) * ((n + edges[i] - 1) / edges[i]);
    // 256-wide tiles run one a CU, in whole rounds
    const double load = i == 2 ? (double)((t + 255) / 256) : t / 256.0;
    const double us = std::max(least[i], each[i] * load);
    if (!p.edge || us < best) best = us, p.edge = edges[i], tiles = t;
  }
  const int64_t stages = (k + kStage - 1) / kStage;
  p.splits = (int)std::max((int64_t)1, std::min(stages / 12, (p.edge == 64 ? 512 : 256) / tiles));
  return p;
}

template <int WM, int WN, int FM, int FN, int DT>
static int mx_gemm(const MxOperand& a, const MxOperand& b, int k, int splits, void* y, hipStream_t st) {
  constexpr int BM = 16 * WM * FM, BN = 16 * WN * FN, lds = 2 * (BM + BN) * kStageBytes;
  static_assert(WM * WN * FM * FN * 512 <= lds, "the results pass through the staging buffers");
  const int64_t mt = (a.rows + BM - 1) / BM, nt = (b.rows + BN - 1) / BN;
  if (mt > most_workgroups(64 * WM * WN) / nt / splits) return set_error(CP_ERR_SHAPE, "product too large");
  static std::atomic<uint64_t> done{0};
  if (int s = allow_lds(reinterpret_cast<const void*>(&mx4_gemm_kernel<WM, WN, FM, FN, DT>), lds, &done,
                        "LDS of the MXFP4 product"))
    return s;
  mx4_gemm_kernel<WM, WN, FM, FN, DT><<<dim3((unsigned)(mt * nt * splits)), 64 * WM * WN, lds, st>>>(
      a, b, k, (int)mt, (int)nt, splits, (typename Elem<DT>::T*)y);
  CP_LAUNCHED("MXFP4 product");
  return CP_OK;
}

template <int DT>
static int mx_gemm_edge(const MxPlan& p, const MxOperand& a, const MxOperand& b, int k, void* y, hipStream_t st) {
  if (p.edge == 64) return mx_gemm<2, 2, 2, 2, DT>(a, b, k, p.splits, y, st);
  if (p.edge == 128) return mx_gemm<2, 2, 4, 4, DT>(a, b, k, p.splits, y, st);
  return mx_gemm<2, 4, 8, 4, DT>(a, b, k, p.splits, y, st);
}

template <int MT, int NT, int XT, int DT>
static int mx_few(const MxOperand& a, const MxOperand& b, const void* x, int64_t stride, int k, void* y,
                  hipStream_t st) {
  const int64_t wgs = (b.rows + 16 * NT - 1) / (16 * NT);
  if (wgs > most_workgroups(1024)) return set_error(CP_ERR_SHAPE, "product too large");
  // Waves: four (more gain nothing: 1 x 1024 x 4096 3.3, 3.6, 4.2 us with 4, 8 and 16). Where
  // they quantize, more while a thread has over four chunks of eight values and the launch
  // under eight waves a CU (8 x 1024 x 4096 9.4 us with 4, 7.0 with 16).
  int w = kFewWaves;
  if (XT >= 0)
    while (w < 16 && wgs * w < 2048 && a.rows * (k / 8) > 4 * 64 * w) w *= 2;
  size_t lds = (size_t)w * MT * NT * 1024;
  if (XT >= 0) lds = std::max(lds, (size_t)a.rows * (k / 2 + 16 + k / kMxBlock));
  mx4_few_kernel<MT, NT, XT, DT><<<dim3((unsigned)wgs), 64 * w, lds, st>>>(a, b, x, stride, k, (int)wgs,
                                                                      (typename Elem<DT>::T*)y);
  CP_LAUNCHED("MXFP4 product");
  return CP_OK;
}

static size_t mx_product_ws(int64_t m, int64_t n, int64_t k) {
  const MxPlan p = mx_plan(m, n, k);
  return p.splits > 1 ? (size_t)m * n * p.splits * 4 : 0;
}

template <int DT>
static int mx_product(const MxOperand& a, const MxOperand& b, int k, void* y, void* ws, hipStream_t st) {
  const MxPlan p = mx_plan(a.rows, b.rows, k);
  // two tiles of b a workgroup where that still fills the CUs: a's rows are read half as often
  // (one / two: 16 x 8192 x 4096 6.1 / 4.9 us, 16 x 14336 x 4096 10.2 / 7.8, 16 x 4096 x 4096
  // 3.9 / 4.9, 16 x 4096 x 14336 9.5 / 12.7)
  const bool wide = b.rows >= 8192;
  if (p.few == 1)
    return wide ? mx_few<1, 2, -1, DT>(a, b, nullptr, 0, k, y, st) : mx_few<1, 1, -1, DT>(a, b, nullptr, 0, k, y, st);
  if (p.few == 2)
    return wide ? mx_few<2, 2, -1, DT>(a, b, nullptr, 0, k, y, st) : mx_few<2, 1, -1, DT>(a, b, nullptr, 0, k, y, st);
  if (p.splits == 1) return mx_gemm_edge<DT>(p, a, b, k, y, st);
  if (int s = mx_gemm_edge<CP_F32>(p, a, b, k, ws, st)) return s;
  const int64_t count = a.rows * b.rows;
  mx4_join_kernel<DT><<<dim3((unsigned)((count + 1023) / 1024)), 256, 0, st>>>((const float*)ws, count, p.splits,
                                                                              (typename Elem<DT>::T*)y);
  CP_LAUNCHED("MXFP4 product's join");
  return CP_OK;
}

// Few rows are quantized inside the product: every workgroup makes the codes for itself, beside
// its first loads of b. GPU time fused / in a launch before it: 4 rows x 1000 x 1056 4.3 / 5.2
// us, 16 5.6 / 5.3, 1 x 4096 x 4096 4.4 / 5.5, 4 5.6 / 5.6, 8 7.2 / 5.8, 1 x 14336 x 4096 8.6 /
// 8.9, 2 9.8 / 9.0: even where a workgroup's share m k reaches 2^14 values or all workgroups'
// m k n 2^26. The second launch also costs the host 4 us, so the bounds are a little above.
static bool mx_fuses(int64_t m, int64_t n, int64_t k) {
  return m <= 32 && m * k <= 24576 && m * k * n <= ((int64_t)1 << 27);
}

template <int XT>
static int mx_fused(const void* x, int64_t m, int64_t stride, const MxOperand& b, int k, void* y, int dt,
                    hipStream_t st) {
  const MxOperand a = {nullptr, nullptr, m};
#define CP_MX_FUSED(DT) \
  return m <= 16 ? mx_few<1, 1, XT, DT>(a, b, x, stride, k, y, st) : mx_few<2, 1, XT, DT>(a, b, x, stride, k, y, st)
  if (dt == CP_F32) CP_MX_FUSED(CP_F32);
  if (dt == CP_BF16) CP_MX_FUSED(CP_BF16);
  CP_MX_FUSED(CP_F16);
#undef CP_MX_FUSED
}

static int mx_launch_product(const MxOperand& a, const MxOperand& b, int k, void* y, int dt, void* ws,
                             hipStream_t st) {
  if (dt == CP_F32) return mx_product<CP_F32>(a, b, k, y, ws, st);
  if (dt == CP_BF16) return mx_product<CP_BF16>(a, b, k, y, ws, st);
  return mx_product<CP_F16>(a, b, k, y, ws, st);
}

static int mx_shape(int64_t rows, int64_t k, const char* what) {
  if (rows < 0 || k <= 0 || k % kMxBlock || k > (1 << 23) || rows > ((int64_t)1 << 40) / k)
    return set_error(CP_ERR_SHAPE, "%s is [%lld, %lld]: rows hold whole blocks of 32 values", what,
                     (long long)rows, (long long)k);
  return CP_OK;
}

static int mx_quantize(const void* x, int dt, int64_t rows, int64_t k, int64_t stride,
                       uint8_t* codes, uint8_t* scales, hipStream_t st) {
  const int64_t groups = mx_groups(rows);
  const unsigned gy = (unsigned)(groups < 65535 ? groups : 65535);
  const int64_t gz = (groups + gy - 1) / gy;
  if (gz > 65535) return set_error(CP_ERR_SHAPE, "too many rows");
  const dim3 grid((unsigned)mx_steps(k), gy, (unsigned)gz);
  if (dt == CP_F32)
    mx4_quantize_kernel<CP_F32><<<grid, 256, 0, st>>>((const float*)x, rows, (int)k, stride, codes, scales);
  if (dt == CP_BF16)
    mx4_quantize_kernel<CP_BF16><<<grid, 256, 0, st>>>((const __bf16*)x, rows, (int)k, stride, codes, scales);
  if (dt == CP_F16)
    mx4_quantize_kernel<CP_F16><<<grid, 256, 0, st>>>((const _Float16*)x, rows, (int)k, stride, codes, scales);
  CP_LAUNCHED("MXFP4 quantize");
  return CP_OK;
}

static int mx_check_x(const void* x, int dt, int64_t rows, int64_t k, int64_t stride) {
  if (int s = mx_shape(rows, k, "x")) return s;
  const int es = dtype_bytes(dt);
  if (!es) return set_error(CP_ERR_ARG, "dtype code %d", dt);
  if (rows > 1 && stride < k) return set_error(CP_ERR_SHAPE, "row stride %lld below %lld", (long long)stride, (long long)k);
  if (rows && !x) return set_error(CP_ERR_ARG, "null x");
  if (!aligned(x, 16) || (rows > 1 && stride * es % 16))
    return set_error(CP_ERR_ALIGN, "rows of x need 16-byte alignment");
  return CP_OK;
}

static int mx_check_ws(const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return set_error(CP_ERR_WORKSPACE, "workspace of %zu bytes needs %zu", have, need);
  if (need && !aligned(ws, 256)) return set_error(CP_ERR_ALIGN, "workspace needs 256-byte alignment");
  return CP_OK;
}

// Bytes of the codes of m rows, a multiple of 256.
static size_t mx_code_bytes(int64_t m, int64_t k) { return (size_t)((m * (k / 2) + 255) / 256 * 256); }

static int mx_check_packed(const uint8_t* codes, const uint8_t* scales, int64_t rows) {
  if (rows && (!codes || !scales)) return set_error(CP_ERR_ARG, "null codes / scales");
  if (!aligned(codes, 16) || !aligned(scales, 4))
    return set_error(CP_ERR_ALIGN, "codes need 16-byte and scales 4-byte alignment");
  return CP_OK;
}

}  // namespace cp

extern "C" {

size_t cp_mx4_scale_bytes(int64_t rows, int64_t k) {
  if (rows < 0 || k < 0) return 0;
  return (size_t)(cp::mx_steps(k) * cp::mx_groups(rows) * 256);
}

int cp_mx4_quantize(const void* x, int x_dtype, int64_t rows, int64_t k, int64_t row_stride,
                    uint8_t* codes, uint8_t* scales, void* stream) {
  cp::clear_error();
  if (int s = cp::mx_check_x(x, x_dtype, rows, k, row_stride)) return s;
  if (int s = cp::mx_check_packed(codes, scales, rows)) return s;
  if (rows == 0) return CP_OK;
  return cp::mx_quantize(x, x_dtype, rows, k, row_stride, codes, scales, (hipStream_t)stream);
}

int cp_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, void* y,
                      int y_dtype, void* stream) {
  cp::clear_error();
  if (int s = cp::mx_shape(rows, k, "y")) return s;
  if (!cp::dtype_bytes(y_dtype)) return cp::set_error(CP_ERR_ARG, "dtype code %d", y_dtype);
  if (int s = cp::mx_check_packed(codes, scales, rows)) return s;
  if (rows && !y) return cp::set_error(CP_ERR_ARG, "null y");
  if (!cp::aligned(y, 16)) return cp::set_error(CP_ERR_ALIGN, "y needs 16-byte alignment");
  if (rows == 0) return CP_OK;
  const int64_t groups = cp::mx_groups(rows);
  const unsigned gy = (unsigned)(groups < 65535 ? groups : 65535);
  const int64_t gz = (groups + gy - 1) / gy;
  if (gz > 65535) return cp::set_error(CP_ERR_SHAPE, "too many rows");
  const dim3 grid((unsigned)cp::mx_steps(k), gy, (unsigned)gz);
  hipStream_t st = (hipStream_t)stream;
  if (y_dtype == CP_F32)
    cp::mx4_dequantize_kernel<CP_F32><<<grid, 256, 0, st>>>(codes, scales, rows, (int)k, (float*)y);
  if (y_dtype == CP_BF16)
    cp::mx4_dequantize_kernel<CP_BF16><<<grid, 256, 0, st>>>(codes, scales, rows, (int)k, (__bf16*)y);
  if (y_dtype == CP_F16)
    cp::mx4_dequantize_kernel<CP_F16><<<grid, 256, 0, st>>>(codes, scales, rows, (int)k, (_Float16*)y);
  CP_LAUNCHED("MXFP4 dequantize");
  return CP_OK;
}

size_t cp_mx4_matmul_ws_bytes(int64_t m, int64_t n, int64_t k) {
  if (m < 1 || n < 1 || k < 1) return 0;
  return cp::mx_product_ws(m, n, k);
}

int cp_mx4_matmul(const uint8_t* a_codes, const uint8_t* a_scales, int64_t m, const uint8_t* b_codes,
                  const uint8_t* b_scales, int64_t n, int64_t k, void* y, int y_dtype, void* ws, size_t ws_bytes,
                  void* stream) {
  cp::clear_error();
  if (int s = cp::mx_shape(m, k, "a")) return s;
  if (int s = cp::mx_shape(n, k, "b")) return s;
  if (!cp::dtype_bytes(y_dtype)) return cp::set_error(CP_ERR_ARG, "dtype code %d", y_dtype);
  if (int s = cp::mx_check_packed(a_codes, a_scales, m)) return s;
  if (int s = cp::mx_check_packed(b_codes, b_scales, n)) return s;
  if (m == 0 || n == 0) return CP_OK;
  if (!y) return cp::set_error(CP_ERR_ARG, "null y");
  if (!cp::aligned(y, 16)) return cp::set_error(CP_ERR_ALIGN, "y needs 16-byte alignment");
  if (int s = cp::mx_check_ws(ws, ws_bytes, cp_mx4_matmul_ws_bytes(m, n, k))) return s;
  return cp::mx_launch_product({a_codes, a_scales, m}, {b_codes, b_scales, n}, (int)k, y, y_dtype, ws,
                               (hipStream_t)stream);
}

size_t cp_mx4_linear_ws_bytes(int64_t m, int64_t n, int64_t k) {
  if (m < 1 || n < 1 || k < 1 || cp::mx_fuses(m, n, k)) return 0;
  return cp::mx_code_bytes(m, k) + cp_mx4_scale_bytes(m, k) + cp_mx4_matmul_ws_bytes(m, n, k);
}

int cp_mx4_linear(const void* x, int x_dtype, int64_t m, int64_t row_stride, const uint8_t* w_codes,
                  const uint8_t* w_scales, int64_t n, int64_t k, void* y, int y_dtype, void* ws,
                  size_t ws_bytes, void* stream) {
  cp::clear_error();
  if (int s = cp::mx_check_x(x, x_dtype, m, k, row_stride)) return s;
  if (int s = cp::mx_shape(n, k, "w")) return s;
  if (!cp::dtype_bytes(y_dtype)) return cp::set_error(CP_ERR_ARG, "dtype code %d", y_dtype);
  if (int s = cp::mx_check_packed(w_codes, w_scales, n)) return s;
  if (m == 0 || n == 0) return CP_OK;
  if (!y) return cp::set_error(CP_ERR_ARG, "null y");
  if (!cp::aligned(y, 16)) return cp::set_error(CP_ERR_ALIGN, "y needs 16-byte alignment");
  if (int s = cp::mx_check_ws(ws, ws_bytes, cp_mx4_linear_ws_bytes(m, n, k))) return s;
  if (cp::mx_fuses(m, n, k)) {
    const cp::MxOperand b = {w_codes, w_scales, n};
    if (x_dtype == CP_F32) return cp::mx_fused<CP_F32>(x, m, row_stride, b, (int)k, y, y_dtype, (hipStream_t)stream);
    if (x_dtype == CP_BF16) return cp::mx_fused<CP_BF16>(x, m, row_stride, b, (int)k, y, y_dtype, (hipStream_t)stream);
    return cp::mx_fused<CP_F16>(x, m, row_stride, b, (int)k, y, y_dtype, (hipStream_t)stream);
  }
  // the rows' codes, their scales, the product's own
  uint8_t* xc = (uint8_t*)ws;
  uint8_t* xs = xc + cp::mx_code_bytes(m, k);
  if (int s = cp::mx_quantize(x, x_dtype, m, k, row_stride, xc, xs, (hipStream_t)stream)) return s;
  return cp::mx_launch_product({xc, xs, m}, {w_codes, w_scales, n}, (int)k, y, y_dtype, xs + cp_mx4_scale_bytes(m, k),
                               (hipStream_t)stream);
}

}  // extern "C"
