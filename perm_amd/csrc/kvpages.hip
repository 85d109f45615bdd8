// The page table of a paged cache kept on the GPU (gfx950): sequences that share pages, pages for
// their next tokens, pages given back, and the pages in use moved to the front.
//
// refs[p] counts the entries of the table that hold page p; a page without holders (refs <= 0)
// is free. Fresh pages are the free ones with the lowest numbers, handed out in the order of
// the sequences and of their entries, so that a call's outcome depends on its inputs alone:
// atomics only add whole numbers, whose order changes nothing.
//
// The books are a few thousand integers, so these kernels are bound by latency (launch, and
// reads that depend on each other); the pages themselves move in kv_copy_kernel, bound by HBM.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kvcache.h"
#include "lowbit.h"

namespace cp {

constexpr int kPagesBlock = 1024;  // pages of one count: 16 a lane

struct Books {
  int* refs;   // [pages]
  int* table;  // [batch][max_pages]
  int pages, batch, max_pages;
};

__device__ __forceinline__ bool is_page(const Books& k, int p) { return (unsigned)p < (unsigned)k.pages; }

// Sum over the wave, in every lane.
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) v += __shfl_xor(v, s);
  return v;
}

// children[i]'s entries become those of parents[i] that its tokens are in, and -1 past them. A
// thread an entry.
__global__ __launch_bounds__(256) void kv_fork_kernel(Books k, const int* lens, int block, const int* parents,
                                                      const int* children, int n) {
  const int chunks = (k.max_pages + 255) / 256;
  const int i = blockIdx.x / chunks, e = (blockIdx.x % chunks) * 256 + threadIdx.x;
  const int from = parents[i], to = children[i];
  if ((unsigned)from >= (unsigned)k.batch || (unsigned)to >= (unsigned)k.batch || from == to || e >= k.max_pages) return;
  const int64_t held = ((int64_t)max(lens[from], 0) + block - 1) / block;
  const int p = e < held ? k.table[(int64_t)from * k.max_pages + e] : -1;
  const bool real = is_page(k, p);
  k.table[(int64_t)to * k.max_pages + e] = real ? p : -1;
  if (real) atomicAdd(k.refs + p, 1);
}

// The entries of these rows (null: of all) become -1, their pages lose a holder each. An entry is
// taken by an exchange, so a row named twice gives its pages back once.
__global__ __launch_bounds__(256) void kv_free_kernel(Books k, const int* rows, int n) {
  const int chunks = (k.max_pages + 255) / 256;
  const int i = blockIdx.x / chunks, e = (blockIdx.x % chunks) * 256 + threadIdx.x;
  const int b = rows ? rows[i] : i;
  if ((unsigned)b >= (unsigned)k.batch || e >= k.max_pages) return;
  int* at = k.table + (int64_t)b * k.max_pages + e;
  if (*at == -1) return;
  const int p = atomicExch(at, -1);
  if (is_page(k, p)) atomicSub(k.refs + p, 1);
}

// Whether page 64 i + lane of block `at` is in use, for i < 16, by bits: one wave, all loads in flight.
// Pages past the last are.
__device__ __forceinline__ uint32_t in_use(const Books& k, int at) {
  const int p0 = at * kPagesBlock + (threadIdx.x & 63);
  int v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = k.refs[min(p0 + 64 * i, k.pages - 1)];
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) bits |= (p0 + 64 * i >= k.pages || v[i] > 0 ? 1u : 0u) << i;
  return bits;
}

__device__ __forceinline__ int count_in_use(const Books& k, int at) {
  return wave_sum(__popc(in_use(k, at))) - max((at + 1) * kPagesBlock - k.pages, 0);
}

// counts[i]: pages of block i in use. A wave a block.
__global__ __launch_bounds__(256) void kv_count_kernel(Books k, int* counts, int blocks) {
  const int at = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= blocks) return;
  const int c = count_in_use(k, at);
  if ((threadIdx.x & 63) == 0) counts[at] = c;
}

struct GrowArgs {
  Books k;
  const int *filled, *fresh;  // [batch]: tokens held, tokens to come (null: `each` of all)
  int each, block;
  int *src, *dst, *missing;   // [batch]
  int* counts;                // [blocks]
  int blocks, counted;
  int *wants, *starts;        // [batch]: pages wanted, and by the sequences before it
  int *pool, *old;            // [pages]: the pages handed out in order, and those they replace
};

// Which entries sequence b needs a page for. first .. last: the entries of its next tokens, of
// which entry `first` holds tokens already if part.
struct GrowRange {
  int64_t first, last;
  bool part, any;
};

__device__ __forceinline__ GrowRange grow_range(const GrowArgs& a, int b) {
  const int64_t held = max(a.filled[b], 0), n = a.fresh ? a.fresh[b] : a.each;
  return {held / a.block, (held + n - 1) / a.block, held % a.block > 0, n > 0};
}

// Whether entry e needs a page: it has none and no tokens, or others hold its page.
__device__ __forceinline__ bool grow_wants(const GrowArgs& a, const GrowRange& g, int64_t e, int p) {
  return is_page(a.k, p) ? a.k.refs[p] > 1 : !(g.part && e == g.first);
}

// f(sequence, its range, this thread's place among the ones that share it and their number, the last of its
// entries in the row): a thread a sequence of up to four entries, as the next token has, then a
// wave a longer one. (A wave for every one, 272 sequences: 46 us, so 12.)
template <class F>
__device__ __forceinline__ void for_sequences(const GrowArgs& a, F f) {
  const int lane = threadIdx.x & 63;
  const int64_t most = a.k.max_pages - 1;
  for (int b0 = 0; b0 < a.k.batch; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    GrowRange g = {};
    int64_t end = -1;
    bool longer = false;
    if (b < a.k.batch) {
      g = grow_range(a, b);
      end = g.any ? min(g.last, most) : g.first - 1;
      longer = end - g.first >= 4;
      if (!longer) f(b, g, 0, 1, end);
    }
    for (unsigned long long left = __ballot(longer); left; left &= left - 1) {
      const int l = __ffsll(left) - 1, c = b0 + (int)(threadIdx.x & ~63u) + l;
      const GrowRange h = grow_range(a, c);
      f(c, h, lane, 64, min(h.last, most));
    }
  }
}

// Sums v over the threads before this one and over all (1024 threads).
template <class T>
__device__ __forceinline__ T scan1024(T v, T* sm, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T sum = v;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const T o = __shfl_up(sum, s);
    if (lane >= s) sum += o;
  }
  if (lane == 63) sm[wave] = sum;
  __syncthreads();
  T base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    base += w < wave ? sm[w] : 0;
    all += sm[w];
  }
  __syncthreads();
  *total = all;
  return base + sum - v;
}

// One workgroup does it all, phase by phase. 1: every sequence's wants. 2: their sums
// in order, and which sequences are served: those up to the first whose sum passes the free pages.
// 3: the free pages in order. 4: entries. 5: holders, once nobody reads them any more.
__global__ __launch_bounds__(1024) void kv_grow_kernel(GrowArgs a) {
  __shared__ int64_t sm[16];
  __shared__ int sm_given;
  const Books& k = a.k;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (!a.counted)
    for (int at = wave; at < a.blocks; at += 16) {
      const int c = count_in_use(k, at);
      if (lane == 0) a.counts[at] = c;
    }
  for_sequences(a, [&](int b, const GrowRange& g, int at, int by, int64_t end) {
    const int* row = k.table + (int64_t)b * k.max_pages;
    int n = 0;
    for (int64_t e = g.first + at; e <= end; e += by) n += grow_wants(a, g, e, row[e]);
    if (by > 1) n = wave_sum(n);
    if (at == 0) {
      a.src[b] = a.dst[b] = -1;
      a.wants[b] = n;
    }
  });
  __syncthreads();
  // free pages in all
  int64_t used = 0, total;
  for (int i = threadIdx.x; i < a.blocks; i += 1024) used += a.counts[i];
  scan1024(used, sm, &total);
  const int64_t free_pages = k.pages - total;
  // the first sequence that is not served ends the sums
  if (threadIdx.x == 0) sm_given = 0;
  int64_t base = 0;
  __syncthreads();
  for (int b0 = 0; b0 < k.batch; b0 += 1024) {
    const int b = b0 + threadIdx.x;
    int64_t n = 0, want = 0, past = 0;  // past: entries past the end of the table
    if (b < k.batch) {
      const GrowRange g = grow_range(a, b);
      n = a.wants[b];
      past = g.any ? max(g.last + 1 - max(g.first, (int64_t)k.max_pages), (int64_t)0) : 0;
      want = past ? 0 : n;
    }
    int64_t sum;
    const int64_t at = base + scan1024(want, sm, &sum);
    if (b < k.batch) {
      const bool got = !past && at + want <= free_pages;
      a.starts[b] = got ? (int)at : -1;
      a.missing[b] = got ? 0 : (int)min(n + past, (int64_t)0x7FFFFFFF);
      if (got && want) atomicMax(&sm_given, (int)(at + want));
    }
    base += sum;
  }
  __syncthreads();
  const int given = sm_given;
  // the first `given` free pages: 64 blocks' counts at a time, a wave a block that has any (294912 pages with
  // the last 300 free: block by block 66 us, so 18)
  int before = 0;
  for (int at0 = 0; at0 < a.blocks && before < given; at0 += 64) {
    const int own = at0 + lane < a.blocks ? min(k.pages - (at0 + lane) * kPagesBlock, kPagesBlock) - a.counts[at0 + lane] : 0;
    int sum = own;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int o = __shfl_up(sum, s);
      if (lane >= s) sum += o;
    }
    for (unsigned long long left = __ballot(own > 0) & 0x0001000100010001ull << wave; left; left &= left - 1) {
      const int l = __ffsll(left) - 1, at = at0 + l;
      int r = before + __shfl(sum - own, l);
      if (r >= given) break;
      const uint32_t bits = in_use(k, at);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool fr = !(bits >> i & 1);
        const unsigned long long m = __ballot(fr);
        const int mine = r + __popcll(m & ((1ull << lane) - 1));
        if (fr && mine < given) a.pool[mine] = at * kPagesBlock + 64 * i + lane;
        r += __popcll(m);
      }
    }
    before += __shfl(sum, 63);
  }
  __syncthreads();
  for_sequences(a, [&](int b, const GrowRange& g, int at, int by, int64_t end) {
    int r = a.starts[b];
    if (r < 0 || a.wants[b] == 0) return;
    int* row = k.table + (int64_t)b * k.max_pages;
    for (int64_t e0 = g.first; e0 <= end; e0 += by) {
      const int64_t e = e0 + at;
      const int p = e <= end ? row[e] : -1;
      const bool w = e <= end && grow_wants(a, g, e, p);
      const unsigned long long m = by > 1 ? __ballot(w) : w;
      const int mine = r + (by > 1 ? __popcll(m & ((1ull << lane) - 1)) : 0);
      if (w) {
        const int q = a.pool[mine];
        row[e] = q;
        a.old[mine] = is_page(k, p) ? p : -1;
        if (g.part && e == g.first) a.src[b] = p, a.dst[b] = q;
      }
      r += __popcll(m);
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < given; i += 1024) {
    k.refs[a.pool[i]] = 1;
    if (a.old[i] >= 0) atomicSub(k.refs + a.old[i], 1);
  }
}

struct CompactArgs {
  Books k;
  int *src, *dst, *used;  // [pages / 2], [pages / 2], [1]
  int* counts;            // [blocks]
  int* rank;              // [pages]: which move takes page p
  int blocks;
};

// The moves: the in-use pages at or past the number in use, in order, go to the free pages before
// it, in order. A workgroup a block of pages; each sums the blocks' counts by itself, and counts
// the pages in use of the block in which that number lies.
__global__ __launch_bounds__(1024) void kv_moves_kernel(CompactArgs a) {
  __shared__ int sm[16];
  const Books& k = a.k;
  int v = 0, used, mine, lower;
  for (int i = threadIdx.x; i < a.blocks; i += 1024) v += a.counts[i];
  scan1024(v, sm, &used);
  v = 0;
  for (int i = threadIdx.x; i < (int)blockIdx.x; i += 1024) v += a.counts[i];
  scan1024(v, sm, &mine);  // in use before this block
  v = 0;
  const int split = used / kPagesBlock;
  for (int i = threadIdx.x; i < split; i += 1024) v += a.counts[i];
  for (int i = split * kPagesBlock + threadIdx.x; i < used; i += 1024) v += k.refs[i] > 0;
  scan1024(v, sm, &lower);  // in use before page `used`
  const int moves = used - lower;
  const int p0 = blockIdx.x * kPagesBlock;
  const int p = p0 + threadIdx.x;
  const bool in = p < k.pages, use = in && k.refs[p] > 0;
  int sum;
  const int before = mine + scan1024((int)use, sm, &sum);
  if (in) {
    if (p >= used) {
      if (use) a.src[before - lower] = p;
      a.rank[p] = use ? before - lower : -1;
    } else if (!use) {
      a.dst[p - before] = p;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.used[0] = used;
  for (int i = moves + blockIdx.x * 1024 + threadIdx.x; i < k.pages / 2; i += a.blocks * 1024) a.src[i] = a.dst[i] = -1;
}

// Entries and holders follow the moves.
__global__ __launch_bounds__(256) void kv_moved_kernel(CompactArgs a) {
  const Books& k = a.k;
  const int used = a.used[0];
  const int64_t entries = (int64_t)k.batch * k.max_pages, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = i0; i < entries; i += (int64_t)gridDim.x * 256) {
    const int p = k.table[i];
    if (!is_page(k, p) || p < used) continue;
    const int r = a.rank[p];
    k.table[i] = r < 0 ? -1 : a.dst[r];
  }
  for (int64_t i = i0; i < k.pages / 2; i += (int64_t)gridDim.x * 256) {
    const int s = a.src[i];
    if (s < 0) continue;
    k.refs[a.dst[i]] = k.refs[s];
    k.refs[s] = 0;
  }
}

struct CopyArgs {
  const uint8_t *k, *v;
  const float *ks, *vs;
  uint8_t *to_k, *to_v;
  float *to_ks, *to_vs;
  const int *src, *dst;
  int pages, to_pages, heads, parts;
  int bytes;  // of a page's codes, K or V
};

constexpr int kCopyPart = 16384;  // bytes of a workgroup

// Page src[i] of one cache into page dst[i] of another or the same one: up to 16 KB of its codes a
// workgroup, four loads of 16 bytes in flight a thread, and the scales with the first. Bound by HBM: 34 MB read and
// written in 11.8 us.
__global__ __launch_bounds__(256) void kv_copy_kernel(CopyArgs a) {
  const int i = blockIdx.x / (2 * a.parts), part = blockIdx.x % (2 * a.parts), at = part >> 1;
  const int s = a.src[i], d = a.dst[i];
  if ((unsigned)s >= (unsigned)a.pages || (unsigned)d >= (unsigned)a.to_pages) return;
  const bool v = part & 1;
  const uint8_t* from = (v ? a.v : a.k) + (int64_t)s * a.bytes;
  uint8_t* to = (v ? a.to_v : a.to_k) + (int64_t)d * a.bytes;
  const int x0 = at * kCopyPart + 16 * threadIdx.x, end = min(a.bytes, (at + 1) * kCopyPart);
  u32x4 w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (x0 + 4096 * j < end) w[j] = *reinterpret_cast<const u32x4*>(from + x0 + 4096 * j);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (x0 + 4096 * j < end) *reinterpret_cast<u32x4*>(to + x0 + 4096 * j) = w[j];
  if (at == 0) {
    const float* fs = (v ? a.vs : a.ks) + (int64_t)s * a.heads;
    float* ts = (v ? a.to_vs : a.to_ks) + (int64_t)d * a.heads;
    for (int h = threadIdx.x; h < a.heads; h += 256) ts[h] = fs[h];
  }
}

static int check_books(const int32_t* refs, int64_t pages, const int32_t* table, int64_t batch, int64_t max_pages) {
  if (pages < 1 || pages > 0x7FFFFFFF - kPagesBlock)
    return set_error(CP_ERR_SHAPE, "%lld pages", (long long)pages);
  if (batch < 0 || batch > 0x7FFFFFF || max_pages < 1 || max_pages > 0x7FFFFFFF / 128)
    return set_error(CP_ERR_SHAPE, "table of %lld rows of %lld pages", (long long)batch, (long long)max_pages);
  if (!refs || (batch && !table)) return set_error(CP_ERR_ARG, "null refs / table");
  if (!aligned(refs, 4) || !aligned(table, 4)) return set_error(CP_ERR_ALIGN, "refs and table need 4-byte alignment");
  return CP_OK;
}

static int check_block(int block) {
  if (block != 16 && block != 32 && block != 64 && block != 128)
    return set_error(CP_ERR_SHAPE, "pages of %d tokens: 16, 32, 64 or 128", block);
  return CP_OK;
}

static int blocks_of(int64_t pages) { return (int)((pages + kPagesBlock - 1) / kPagesBlock); }

// int32s of a workspace, in pieces of 256 bytes.
static int64_t ints(int64_t n) { return (n + 63) / 64 * 64; }

static int check_ws(const void* ws, size_t have, size_t need) {
  if (!ws || have < need) return set_error(CP_ERR_WORKSPACE, "workspace of %zu bytes needs %zu", have, need);
  if (!aligned(ws, 256)) return set_error(CP_ERR_ALIGN, "workspace needs 256-byte alignment");
  return CP_OK;
}

}  // namespace cp

extern "C" {

int cp_kv_fork(int32_t* refs, int64_t pages, int32_t* table, int64_t batch, int64_t max_pages, const int32_t* lens,
               int block, const int32_t* parents, const int32_t* children, int64_t n, void* stream) {
  cp::clear_error();
  if (int s = cp::check_books(refs, pages, table, batch, max_pages)) return s;
  if (int s = cp::check_block(block)) return s;
  const int64_t chunks = (max_pages + 255) / 256;
  if (n < 0 || n > 0x7FFFFFFF || n * chunks > cp::most_workgroups(256))
    return cp::set_error(CP_ERR_SHAPE, "%lld forks of %lld pages", (long long)n, (long long)max_pages);
  if (n == 0 || batch == 0) return CP_OK;
  if (!lens || !parents || !children) return cp::set_error(CP_ERR_ARG, "null lens / parents / children");
  const cp::Books k = {refs, table, (int)pages, (int)batch, (int)max_pages};
  cp::kv_fork_kernel<<<dim3((unsigned)(n * chunks)), 256, 0, (hipStream_t)stream>>>(k, lens, block, parents, children,
                                                                                    (int)n);
  CP_LAUNCHED("fork");
  return CP_OK;
}

int cp_kv_free(int32_t* refs, int64_t pages, int32_t* table, int64_t batch, int64_t max_pages, const int32_t* rows,
               int64_t n, void* stream) {
  cp::clear_error();
  if (int s = cp::check_books(refs, pages, table, batch, max_pages)) return s;
  if (!rows) n = batch;
  const int64_t chunks = (max_pages + 255) / 256;
  if (n < 0 || n > 0x7FFFFFFF || n * chunks > cp::most_workgroups(256))
    return cp::set_error(CP_ERR_SHAPE, "%lld rows of %lld pages", (long long)n, (long long)max_pages);
  if (n == 0 || batch == 0) return CP_OK;
  const cp::Books k = {refs, table, (int)pages, (int)batch, (int)max_pages};
  cp::kv_free_kernel<<<dim3((unsigned)(n * chunks)), 256, 0, (hipStream_t)stream>>>(k, rows, (int)n);
  CP_LAUNCHED("free");
  return CP_OK;
}

size_t cp_kv_grow_ws_bytes(int64_t pages, int64_t batch) {
  if (pages < 1 || batch < 1) return 0;
  return 4 * (size_t)(cp::ints(cp::blocks_of(pages)) + 2 * cp::ints(batch) + 2 * cp::ints(pages));
}

int cp_kv_grow(int32_t* refs, int64_t pages, int32_t* table, int64_t batch, int64_t max_pages, const int32_t* filled,
               const int32_t* fresh, int each, int block, int32_t* src, int32_t* dst, int32_t* missing, void* ws,
               size_t ws_bytes, void* stream) {
  cp::clear_error();
  if (int s = cp::check_books(refs, pages, table, batch, max_pages)) return s;
  if (int s = cp::check_block(block)) return s;
  if (batch == 0) return CP_OK;
  if (!filled || !src || !dst || !missing)
    return cp::set_error(CP_ERR_ARG, "null filled / src / dst / missing");
  if (int s = cp::check_ws(ws, ws_bytes, cp_kv_grow_ws_bytes(pages, batch))) return s;
  cp::GrowArgs a;
  a.k = {refs, table, (int)pages, (int)batch, (int)max_pages};
  a.filled = filled;
  a.fresh = fresh;
  a.each = each;
  a.block = block;
  a.src = src;
  a.dst = dst;
  a.missing = missing;
  a.blocks = cp::blocks_of(pages);
  a.counts = (int*)ws;
  a.wants = a.counts + cp::ints(a.blocks);
  a.starts = a.wants + cp::ints(batch);
  a.pool = a.starts + cp::ints(batch);
  a.old = a.pool + cp::ints(pages);
  a.counted = a.blocks > 16;
  if (a.counted) {
    cp::kv_count_kernel<<<dim3((unsigned)((a.blocks + 3) / 4)), 256, 0, (hipStream_t)stream>>>(a.k, a.counts, a.blocks);
    CP_LAUNCHED("page counts");
  }
  cp::kv_grow_kernel<<<dim3(1), 1024, 0, (hipStream_t)stream>>>(a);
  CP_LAUNCHED("grow");
  return CP_OK;
}

size_t cp_kv_compact_ws_bytes(int64_t pages) {
  if (pages < 1) return 0;
  return 4 * (size_t)(cp::ints(cp::blocks_of(pages)) + cp::ints(pages));
}

int cp_kv_compact(int32_t* refs, int64_t pages, int32_t* table, int64_t batch, int64_t max_pages, int32_t* src,
                  int32_t* dst, int32_t* used, void* ws, size_t ws_bytes, void* stream) {
  cp::clear_error();
  if (int s = cp::check_books(refs, pages, table, batch, max_pages)) return s;
  if (!used || (pages > 1 && (!src || !dst))) return cp::set_error(CP_ERR_ARG, "null src / dst / used");
  if (int s = cp::check_ws(ws, ws_bytes, cp_kv_compact_ws_bytes(pages))) return s;
  cp::CompactArgs a;
  a.k = {refs, table, (int)pages, (int)batch, (int)max_pages};
  a.src = src;
  a.dst = dst;
  a.used = used;
  a.blocks = cp::blocks_of(pages);
  a.counts = (int*)ws;
  a.rank = a.counts + cp::ints(a.blocks);
  hipStream_t st = (hipStream_t)stream;
  cp::kv_count_kernel<<<dim3((unsigned)((a.blocks + 3) / 4)), 256, 0, st>>>(a.k, a.counts, a.blocks);
  CP_LAUNCHED("page counts");
  cp::kv_moves_kernel<<<dim3((unsigned)a.blocks), 1024, 0, st>>>(a);
  CP_LAUNCHED("moves");
  const int64_t items = std::max(batch * max_pages, pages / 2);
  if (items == 0) return CP_OK;  // one page and no entries
  cp::kv_moved_kernel<<<dim3((unsigned)std::min((items + 255) / 256, (int64_t)2048)), 256, 0, st>>>(a);
  CP_LAUNCHED("moved entries");
  return CP_OK;
}

int cp_kv_copy(const cp_kv_cache* from, const cp_kv_cache* to, const int32_t* src, const int32_t* dst, int64_t n,
               void* stream) {
  cp::clear_error();
  if (int s = cp::kv_check_cache(from)) return s;
  if (int s = cp::kv_check_cache(to)) return s;
  if (from->heads != to->heads || from->block != to->block || from->head_dim != to->head_dim)
    return cp::set_error(CP_ERR_SHAPE, "pages of %d heads of %d, %d tokens, into pages of %d heads of %d, %d tokens",
                         from->heads, from->head_dim, from->block, to->heads, to->head_dim, to->block);
  cp::CopyArgs a;
  const int64_t bytes = (int64_t)from->heads * from->block * from->head_dim;  // under 2^31
  a.bytes = (int)bytes;
  a.parts = (int)((bytes + cp::kCopyPart - 1) / cp::kCopyPart);
  if (n < 0 || n > 0x7FFFFFFF || n * 2 * a.parts > cp::most_workgroups(256))
    return cp::set_error(CP_ERR_SHAPE, "%lld pages to copy", (long long)n);
  if (n == 0) return CP_OK;
  if (!src || !dst) return cp::set_error(CP_ERR_ARG, "null src / dst");
  a.k = from->k, a.v = from->v, a.ks = from->k_scale, a.vs = from->v_scale;
  a.to_k = to->k, a.to_v = to->v, a.to_ks = to->k_scale, a.to_vs = to->v_scale;
  a.src = src, a.dst = dst;
  a.pages = (int)from->pages, a.to_pages = (int)to->pages, a.heads = from->heads;
  cp::kv_copy_kernel<<<dim3((unsigned)(n * 2 * a.parts)), 256, 0, (hipStream_t)stream>>>(a);
  CP_LAUNCHED("page copy");
  return CP_OK;
}

}  // extern "C"
