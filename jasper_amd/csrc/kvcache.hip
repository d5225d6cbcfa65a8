// kvcache.hip -- rotary positions, appending to the paged cache, and copying
// its pages.
#include "kvcache.hpp"

#include "graph.hpp"
#include "kvtypes.hpp"

#include <algorithm>
#include <stdexcept>

namespace jasper_amd {

namespace {

// One launch turns the heads of q and k and, when APPEND, writes k and v to
// the cache. The heads of a token are one list: q's, then k's, then v's.
struct TokenParams {
  const char *q, *k, *v;
  int64_t q_stride, q_head, k_stride, k_head, v_stride, v_head;
  int q_heads, k_heads, v_heads;
  const void* positions;
  const void* slots;
  const float *cos, *sin;
  int64_t n, table_rows;
  int dim, half;
  bool pos64, slots64, interleaved, back;
  char *q_out, *k_out;
  KvPages pages;
  int64_t rows;  // of the cache: pages * page size
};

__device__ __forceinline__ int64_t index_at(const void* p, bool wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// x / d, with r = 1 / d rounded to nearest: one correction of x * r by its
// exact remainder gives the quotient rounded to nearest (Markstein 1990),
// short of under- and overflow; where x * r is too large for the cache, or not
// finite, it is taken as it is, and so is a zero, which keeps its sign. Three
// operations instead of the ten of a division: 6007 tokens of 8 heads into an
// e4m3 cache 38.7 -> 31.8 us.
__device__ __forceinline__ float quotient(float x, float d, float r) {
  const float q = x * r;
  const float fixed = __builtin_fmaf(__builtin_fmaf(-q, d, x), r, q);
  return __builtin_fabsf(q) < 1e6f && q != 0.f ? fixed : q;
}

// Of quotients from 2^-11 (an e4m3 cache rounds smaller ones to zero) to 1e6
// by such a divisor the remainder above is a number of steps of 2^-137 at
// least, so it is exact; others are divided by.
__device__ __forceinline__ bool quotient_fits(float d) {
  return __builtin_fabsf(d) > 0x1p-80f && __builtin_fabsf(d) < 0x1p80f;
}

// A thread has one chunk of 2 * P values of a head (threadIdx.x) and walks
// the heads of its token (threadIdx.y on) with the chunk's P cosines and
// sines in registers. In the half layout the chunk is P values of each half,
// otherwise 2 * P neighbours; the unrotated tail is chunks of neighbours.
// The products and sums are rounded one by one (no fused multiply-add): the
// same bits as the formula in fp32 operations. Bound by memory: 8192 tokens of
// 32 + 8 heads of 128 bf16 values 38 us (4.4 TB/s read and written; a large copy
// 4.7), 6007 of 32 + 2 x 8 into e4m3 pages 32 us (4.3); one token 3.6 us.
template <typename T, typename CT, int P, bool APPEND>
__global__ void token_kernel(TokenParams a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.z + threadIdx.z;
  if (i >= a.n) return;
  const int c = threadIdx.x, turned = a.half / P;
  const bool turn = c < turned;
  const bool split = turn && !a.interleaved;
  const int at = split ? c * P : c * 2 * P;
  const int to = split ? a.half + at : at + P;
  float co[P], si[P];
  if (turn) {
    const int64_t pos = index_at(a.positions, a.pos64, i);
    const bool known = pos >= 0 && pos < a.table_rows;
    const int64_t row = known ? pos * a.half + c * P : 0;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      co[e] = known ? a.cos[row + e] : __builtin_nanf("");
      si[e] = known ? (a.back ? -a.sin[row + e] : a.sin[row + e]) : __builtin_nanf("");
    }
  }
  int64_t slot = -1;
  if (APPEND) slot = index_at(a.slots, a.slots64, i);
  const bool kept = APPEND && slot >= 0 && slot < a.rows;
  const int64_t page = kept ? slot >> a.pages.page_shift : 0;
  const int64_t in_page = kept ? slot & (a.pages.page - 1) : 0;
  const int all = a.q_heads + a.k_heads + a.v_heads;
  for (int h = blockIdx.y * blockDim.y + threadIdx.y; h < all; h += blockDim.y * gridDim.y) {
    const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.k_heads;
    const int hh = is_q ? h : is_v ? h - a.q_heads - a.k_heads : h - a.q_heads;
    if (APPEND && !is_q && !kept) continue;
    const T* src = (const T*)(is_q ? a.q : is_v ? a.v : a.k) +
                   (is_q ? i * a.q_stride + hh * a.q_head : is_v ? i * a.v_stride + hh * a.v_head
                                                                 : i * a.k_stride + hh * a.k_head);
    // v is not rotated: its chunks are neighbours
    const int from = is_v ? c * 2 * P : at, other = is_v ? c * 2 * P + P : to;
    float x[2 * P];
    widen(*(const Pack<T, P>*)(src + from), x);
    widen(*(const Pack<T, P>*)(src + other), x + P);
    if (turn && !is_v) {
#pragma unroll
      for (int e = 0; e < P; ++e) {
        float& u = a.interleaved ? x[2 * e] : x[e];
        float& w = a.interleaved ? x[2 * e + 1] : x[P + e];
        const float u0 = u, w0 = w;
        u = u0 * co[e] - w0 * si[e];
        w = w0 * co[e] + u0 * si[e];
      }
    }
    if (!APPEND || is_q) {
      T* dst = (T*)(is_q ? a.q_out : a.k_out) + (i * (is_q ? a.q_heads : a.k_heads) + hh) * a.dim;
      *(Pack<T, P>*)(dst + from) = narrow<T, P>(x);
      *(Pack<T, P>*)(dst + other) = narrow<T, P>(x + P);
    } else {
      const float* scales = is_v ? a.pages.v_scale : a.pages.k_scale;
      if (sizeof(CT) == 1 && scales) {
        const float scale = scales[hh], inverse = 1.f / scale;
        if (quotient_fits(scale)) {
#pragma unroll
          for (int e = 0; e < 2 * P; ++e) x[e] = quotient(x[e], scale, inverse);
        } else {
#pragma unroll
          for (int e = 0; e < 2 * P; ++e) x[e] = x[e] / scale;
        }
      }
      CT* dst = (CT*)(is_v ? a.pages.v : a.pages.k) + page * a.pages.page_stride + hh * a.pages.head_stride +
                in_page * a.pages.row_stride;
      *(Pack<CT, P>*)(dst + from) = narrow<CT, P>(x);
      *(Pack<CT, P>*)(dst + other) = narrow<CT, P>(x + P);
    }
  }
}

template <typename T, typename CT, bool APPEND>
void launch_token(const TokenParams& p, int P, hipStream_t s) {
  const int all = p.q_heads + p.k_heads + p.v_heads;
  if (p.n == 0 || all == 0) return;
  const int chunks = p.dim / (2 * P);
  if (chunks > 1024) throw std::invalid_argument("a head is too large");
  // A thread per chunk of a head where that is all there is to do; with more,
  // threads keep their cosines for several heads, up to 12: 512 work-items for
  // each compute unit come first. 445 tokens of 64 + 2 x 8 heads of 256 values
  // 14.4 us (25.3 with a thread each), 6007 of 32 + 2 x 8 of 128 31.5 (33.4 with
  // 10 heads to a thread, 43.8 with 24).
  const int64_t items = p.n * all * chunks;
  const int per = (int)std::clamp<int64_t>(items / 131072, 1, 12), lanes = (all + per - 1) / per;
  dim3 block(chunks, std::min(lanes, std::max(1, 256 / chunks)), 1), grid;
  grid.y = (lanes + block.y - 1) / block.y;
  if (grid.y == 1) block.z = std::max(1u, 256u / (block.x * block.y));
  const int64_t blocks = (p.n + block.z - 1) / block.z;
  if (blocks > 0x7FFFFFFF) throw std::invalid_argument("too many tokens (too large)");
  grid.x = (unsigned)blocks;
  auto kernel = P == 8 ? token_kernel<T, CT, 8, APPEND> : P == 4 ? token_kernel<T, CT, 4, APPEND>
                                                                 : token_kernel<T, CT, 1, APPEND>;
  kernel<<<grid, block, 0, s>>>(p);
  hip_check(hipGetLastError(), "rotary");
}

bool rows_fit(const void* p, int64_t stride, int64_t head_stride, int heads, int width, int bytes) {
  const int64_t unit = (int64_t)width * bytes;
  return heads == 0 || ((uintptr_t)p % (uintptr_t)unit == 0 && stride * bytes % unit == 0 && head_stride * bytes % unit == 0);
}

TokenParams token_params(const RotaryArgs& a) {
  TokenParams p{};
  p.q = (const char*)a.q.p, p.q_stride = a.q.stride, p.q_head = a.q.head_stride, p.q_heads = a.q.heads;
  p.k = (const char*)a.k.p, p.k_stride = a.k.stride, p.k_head = a.k.head_stride, p.k_heads = a.k.heads;
  p.positions = a.positions, p.pos64 = a.pos64, p.cos = a.cos, p.sin = a.sin, p.n = a.n, p.table_rows = a.table_rows;
  p.dim = a.dim, p.half = a.half, p.interleaved = a.interleaved, p.back = a.back;
  return p;
}

// The widest chunks that the sizes, strides and addresses allow.
int chunk_of(const TokenParams& p, int type) {
  const int rest = p.dim - 2 * p.half;
  for (int P : {8, 4}) {
    if (p.half % P || rest % (2 * P)) continue;
    const int b = kv_bytes(type);
    if (rows_fit(p.q, p.q_stride, p.q_head, p.q_heads, P, b) && rows_fit(p.k, p.k_stride, p.k_head, p.k_heads, P, b) &&
        rows_fit(p.v, p.v_stride, p.v_head, p.v_heads, P, b))
      return P;
  }
  return 1;
}

}  // namespace

void rotary(const RotaryArgs& a, void* q_out, void* k_out, hipStream_t s) {
  TokenParams p = token_params(a);
  p.q_out = (char*)q_out, p.k_out = (char*)k_out;
  const int P = chunk_of(p, a.type);
  if (a.type == kF16) launch_token<f16, f16, false>(p, P, s);
  else launch_token<bf16, bf16, false>(p, P, s);
}

void append_tokens(const RotaryArgs& a, const HeadRows& v, const void* slots, bool slots64, const KvPages& pages,
                   void* q_out, hipStream_t s) {
  TokenParams p = token_params(a);
  p.v = (const char*)v.p, p.v_stride = v.stride, p.v_head = v.head_stride, p.v_heads = v.heads;
  p.slots = slots, p.slots64 = slots64, p.pages = pages, p.q_out = (char*)q_out;
  p.rows = (int64_t)pages.pages * pages.page;
  const int P = chunk_of(p, a.type);
  if (pages.type == kE4M3) {
    if (a.type == kF16) launch_token<f16, e4m3, true>(p, P, s);
    else launch_token<bf16, e4m3, true>(p, P, s);
  } else if (a.type == kF16) {
    launch_token<f16, f16, true>(p, P, s);
  } else {
    launch_token<bf16, bf16, true>(p, P, s);
  }
}

// ---- copying pages ----

namespace {

constexpr int kCopyThreads = 256, kCopyUnits = 4;  // 16-byte units a thread moves

struct CopyParams {
  char *k, *v;
  int64_t layer_bytes, page_bytes, head_bytes, row_bytes;
  int pages, page;
  uint32_t units, row_units;  // of a page, of a row
  const int32_t *src, *dst;
  uint32_t n;
  uint32_t moves;        // pages in all: of K and V of every layer
  uint32_t copy_groups;  // of the grid; the rest rewrite table entries
  int32_t* tables;
  int64_t entries;
};

constexpr int kEntries = 64, kSources = 1024;  // table entries of a work-group, sources it holds at once

// Table entries that are sources become destinations: a lane has an entry,
// the four waves a quarter of the sources each. 1,500 small pages with 5,900
// entries: 8.2 us a call, 75 with a thread for each entry and all sources.
__device__ void move_entries(const CopyParams& a, int64_t group) {
  __shared__ __attribute__((aligned(16))) int32_t from[kSources];
  __shared__ int32_t found[kEntries];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t e = group * kEntries + lane;
  const int32_t old = e < a.entries ? a.tables[e] : -1;
  for (uint32_t b = 0; b < a.n; b += kSources) {
    const int m = min(a.n - b, (uint32_t)kSources);
    for (int j = threadIdx.x; j < kSources; j += kCopyThreads) {
      int32_t f = -1;
      if (j < m) {
        const int32_t t = a.dst[b + j];
        f = a.src[b + j];
        if (f >= a.pages || t < 0 || t >= a.pages) f = -1;
      }
      from[j] = f;
    }
    if (threadIdx.x < kEntries) found[threadIdx.x] = -1;
    __syncthreads();
    int32_t hit = -1;
    const int per = kSources / (kCopyThreads / 64);
#pragma unroll 4
    for (int j = wave * per; j < wave * per + per; j += 4) {
      typedef int32_t intx4 __attribute__((ext_vector_type(4)));
      const intx4 f = *(const intx4*)(from + j);
#pragma unroll
      for (int k = 0; k < 4; ++k) hit = f[k] == old ? j + k : hit;
    }
    if (old >= 0 && hit >= 0) found[lane] = hit;  // a source is listed once
    __syncthreads();
    if (wave == 0 && old >= 0 && found[lane] >= 0) a.tables[e] = a.dst[b + found[lane]];
    __syncthreads();
  }
}

// A work-group moves 16 KB, of one page or of several: a thread's four
// 16-byte loads go out before its stores. WHOLE: a page is whole such runs.
// Bound by memory: 513 pages of 16 layers, 64 KB of K and V each, 215 us (5.0
// TB/s read and written; a large copy runs at 4.7). Eight loads per thread
// took 510 us. Four pages of 32 layers 4.4 us, a launch.
template <bool FLAT, bool WHOLE>
__global__ __launch_bounds__(kCopyThreads) void copy_kernel(CopyParams a) {
  if (blockIdx.x >= a.copy_groups) return move_entries(a, blockIdx.x - a.copy_groups);
  constexpr uint32_t kRun = kCopyThreads * kCopyUnits;
  const uint32_t begin = blockIdx.x * kRun, first = begin / a.units, rest = begin % a.units;
  const uint32_t plane0 = first / a.n, pair0 = first % a.n;  // plane: layer and K or V
  uintx4 x[kCopyUnits];
  char* to[kCopyUnits];
#pragma unroll
  for (int j = 0; j < kCopyUnits; ++j) {
    to[j] = nullptr;
    uint32_t u = rest + j * kCopyThreads + threadIdx.x;
    uint32_t plane = plane0, i = pair0;
    if (!WHOLE) {
      const uint32_t k = u / a.units, next = pair0 + k;
      if (first + k >= a.moves) continue;
      u -= k * a.units;
      plane += next / a.n, i = next % a.n;
    }
    const int32_t f = a.src[i], t = a.dst[i];
    if (f < 0 || f >= a.pages || t < 0 || t >= a.pages) continue;
    char* base = (plane & 1 ? a.v : a.k) + (int64_t)(plane >> 1) * a.layer_bytes;
    int64_t off = (int64_t)u * 16;
    if (!FLAT) {
      const uint32_t row = u / a.row_units;
      off = (int64_t)(row / a.page) * a.head_bytes + (int64_t)(row % a.page) * a.row_bytes +
            (int64_t)(u % a.row_units) * 16;
    }
    x[j] = *(const uintx4*)(base + f * a.page_bytes + off);
    to[j] = base + t * a.page_bytes + off;
  }
#pragma unroll
  for (int j = 0; j < kCopyUnits; ++j)
    if (to[j]) *(uintx4*)to[j] = x[j];
}

}  // namespace

void copy_pages(const KvPages& pages, const int32_t* src, const int32_t* dst, int64_t n, int32_t* tables,
                int64_t table_entries, hipStream_t s) {
  if (n == 0) return;
  const int b = kv_bytes(pages.type);
  CopyParams p{};
  p.k = pages.k, p.v = pages.v;
  p.layer_bytes = pages.layer_stride * b, p.page_bytes = pages.page_stride * b;
  p.head_bytes = pages.head_stride * b, p.row_bytes = pages.row_stride * b;
  p.pages = pages.pages, p.page = pages.page;
  p.row_units = (uint32_t)(pages.dim * b / 16);
  const int64_t units = (int64_t)pages.heads * pages.page * p.row_units, run = kCopyThreads * kCopyUnits;
  // as many pairs to a launch as 32 bits count the units of: 32 GB
  const int64_t most = ((int64_t)1 << 31) / std::max<int64_t>(1, 2 * pages.layers * units);
  if (most < 1) throw std::invalid_argument("a page of all layers is too large");
  p.units = (uint32_t)units;
  p.tables = tables, p.entries = tables ? table_entries : 0;
  const int64_t entry_groups = (p.entries + kEntries - 1) / kEntries;
  if (entry_groups > 0x40000000) throw std::invalid_argument("too many table entries (too large)");
  const bool flat = pages.row_stride == pages.dim && pages.head_stride == (int64_t)pages.page * pages.dim;
  const bool whole = units % run == 0;
  auto kernel = flat ? (whole ? copy_kernel<true, true> : copy_kernel<true, false>)
                     : (whole ? copy_kernel<false, true> : copy_kernel<false, false>);
  for (int64_t at = 0; at < n; at += most) {
    p.src = src + at, p.dst = dst + at, p.n = (uint32_t)std::min(most, n - at);
    p.moves = 2 * pages.layers * p.n;
    p.copy_groups = (uint32_t)(((int64_t)p.moves * units + run - 1) / run);
    kernel<<<p.copy_groups + (unsigned)entry_groups, kCopyThreads, 0, s>>>(p);
    hip_check(hipGetLastError(), "copy pages");
  }
}

}  // namespace jasper_amd
