// pagetable.hip -- the page tables of a cache whose bookkeeping is on the GPU.
//
// Which page goes where follows from the state and the request alone: the
// lowest free pages, to the requests in order. Atomic operations only count
// and set bits, so their order changes nothing.
#include "pagetable.hpp"

#include "graph.hpp"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace jasper_amd {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of the planning work-group
constexpr int kRowThreads = 256;
constexpr int kGrowers = 4096;         // last pages held in LDS at once
// Words of the bitmap whose pages waves give out, what LDS holds numbers of; those
// of more are gone through by a thread each: 20,000 pages and their truncation 33.6 us
// in a cache of 262,144, 44.9 in one of 262,176, 162 in one of 2,000,000.
constexpr int kBases = 8192;
constexpr int kSequences = 1 << 18;    // at most: a bit for each in LDS

// What the plan says of a request. fresh: the places of the table from which on
// it gets pages of the list, from place `offset` of it on.
struct Request {
  int32_t seq, from, to, fresh, last;
  int32_t offset, start, count;
  int32_t owners;  // of the page that it grows in
};

struct Extend {
  PageState state;
  const int32_t *seqs, *counts;
  int n, width;
  int64_t n_tokens;
  int64_t *positions, *slots;
  int32_t *starts, *step_tables, *step_lens, *src, *dst, *missing;
  Request* requests;
  int32_t* list;     // the pages given out, in order
  int32_t* growers;  // the last pages of requests that share theirs
};

// x of the lane that DPP control `ctrl` names, 0 where there is none.
template <int ctrl, int rows>
__device__ __forceinline__ int64_t moved(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), ctrl, rows, 0xF, false);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The sum of x over the lanes up to this one, without LDS: rows of 16 lanes
// shifted by 1, 2, 4 and 8, then a row's last lane to the next one and lane 31
// to the last two.
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
  x += moved<0x111, 0xF>(x);
  x += moved<0x112, 0xF>(x);
  x += moved<0x114, 0xF>(x);
  x += moved<0x118, 0xF>(x);
  x += moved<0x142, 0xA>(x);
  x += moved<0x143, 0xC>(x);
  return x;
}

// For N numbers at once: their sums over the threads before this one, and over
// all. `part` has room for N * kWaves numbers and is free again after the next
// barrier.
template <int N>
__device__ __forceinline__ void block_scan(const int64_t (&x)[N], int64_t (&before)[N], int64_t (&total)[N], int64_t* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    before[k] = wave_scan(x[k]);
    if (lane == 63) part[k * kWaves + wave] = before[k];
    before[k] -= x[k];
  }
  __syncthreads();
  const int w = __builtin_amdgcn_readfirstlane(wave);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    // the waves' sums, summed up by the lanes of a row
    int64_t x = part[k * kWaves + (lane & (kWaves - 1))];
    x += moved<0x111, 0xF>(x);
    x += moved<0x112, 0xF>(x);
    x += moved<0x114, 0xF>(x);
    x += moved<0x118, 0xF>(x);
    const auto of = [&](int l) {
      return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, l));
    };
    total[k] = of(kWaves - 1);
    if (w) before[k] += of(w - 1);
  }
}

__device__ __forceinline__ int pages_of(int tokens, int shift) { return (int)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

struct PlanLds {
  alignas(16) int32_t held[kGrowers];  // read four at a time
  int32_t bases[kBases];  // free pages before each word of the bitmap
  int64_t part[5 * kWaves];
};
static_assert(alignof(PlanLds) == 16, "dynamic LDS beside it gives no alignment");

// One work-group decides: how many pages each request takes, which are free,
// whether there are enough. A thread has a run of requests (one of them, in
// registers, where ONE) and a run of the bitmap's words, so that ranks in order
// are ranks of threads. Bound by its chain of dependent loads (sequence, length,
// last page, its owners) and two sums over the work-group: 48 next tokens 6.6 us,
// 256 forks that grow in 64 shared pages 12.6, 700 prompts of 337,000 tokens 17.9.
template <bool ONE>
__device__ void plan(const Extend& a, uint32_t* seen, PlanLds& l) {
  const PageState& st = a.state;
  const int t = threadIdx.x, page = 1 << st.page_shift;
  const int run = ONE ? 1 : (a.n + kThreads - 1) / kThreads, r0 = min(t * run, a.n), r1 = min(r0 + run, a.n);
  Request one{};
  const auto get = [&](int i) -> Request { return ONE ? one : a.requests[i]; };
  const auto put = [&](int i, const Request& q) {
    if (ONE) one = q;
    else a.requests[i] = q;
  };
  // the bitmap's words, on their way while the requests are looked at
  const int words = (st.pages + 31) / 32, wrun = (words + kThreads - 1) / kThreads;
  const int w0 = min(t * wrun, words), w1 = min(w0 + wrun, words);
  const auto word = [&](int w) {
    const uint32_t x = st.free[w];
    return w == words - 1 && (st.pages & 31) ? x & ((1u << (st.pages & 31)) - 1) : x;
  };
  constexpr int kFirst = 4;
  uint32_t early[kFirst];
#pragma unroll
  for (int k = 0; k < kFirst; ++k) early[k] = w0 + k < w1 ? word(w0 + k) : 0;

  for (int i = t; i < (st.sequences + 31) / 32; i += kThreads) seen[i] = 0;
  __syncthreads();
  int64_t growing[1] = {0}, at[1], n_growing[1];
  bool bad = false;
  for (int i = r0; i < r1; ++i) {
    Request q{};
    const int32_t count = a.counts[i];
    q.seq = a.seqs[i], q.last = -1;
    if (q.seq < 0 || q.seq >= st.sequences) {
      q.seq = -1;
    } else {
      const uint32_t bit = 1u << (q.seq & 31);
      bad |= count < 0 || (atomicOr(&seen[q.seq >> 5], bit) & bit);
      q.count = max(count, 0);
      const int64_t most = (int64_t)st.width << st.page_shift;
      q.from = (int32_t)min((int64_t)max(st.lens[q.seq], 0), most);
      bad |= (int64_t)q.from + q.count > min(most, (int64_t)a.width << st.page_shift);
      if (bad) q.count = 0;
      q.to = q.from + q.count;
      q.fresh = pages_of(q.from, st.page_shift);
      if (q.count && (q.from & (page - 1))) {
        const int32_t last = st.tables[(int64_t)q.seq * st.width + q.fresh - 1];
        if (last >= 0 && last < st.pages) {
          q.owners = st.refs[last];
          if (q.owners > 1) q.last = last, ++growing[0];
        }
      }
    }
    put(i, q);
  }
  // requests that share the page they grow in: each copies it, but for the last owner
  block_scan<1>(growing, at, n_growing, l.part);
  if (n_growing[0]) {
    int64_t mine = at[0];
    for (int i = r0; i < r1; ++i) {
      const int32_t last = get(i).last;
      if (last >= 0) a.growers[mine++] = last;
    }
    __syncthreads();
    for (int64_t c = 0; c < n_growing[0]; c += kGrowers) {
      const int m = (int)min((int64_t)kGrowers, n_growing[0] - c);
      for (int i = t; i < (m + 3) / 4 * 4; i += kThreads) l.held[i] = i < m ? a.growers[c + i] : -1;
      __syncthreads();
      mine = at[0];
      for (int i = r0; i < r1; ++i) {
        Request q = get(i);
        if (q.last < 0) continue;
        // those before it that have the same page, four at a time
        const int end = (int)max((int64_t)0, min((int64_t)m, mine - c));
        int before = 0;
        typedef int32_t intx4 __attribute__((ext_vector_type(4)));
#pragma unroll 8
        for (int j = 0; j < end; j += 4) {
          const intx4 h = *(const intx4*)(l.held + j);
#pragma unroll
          for (int k = 0; k < 4; ++k) before += h[k] == q.last && j + k < end;
        }
        q.offset += before;
        put(i, q);
        ++mine;
      }
      __syncthreads();
    }
  }
  int64_t sums[4] = {0, 0, 0, bad}, before[4], total[4];  // pages taken, tokens, free pages, what cannot be
  for (int i = r0; i < r1; ++i) {
    Request q = get(i);
    if (q.last >= 0) {
      if (q.owners - q.offset > 1) --q.fresh;
      else q.last = -1;
      put(i, q);
    }
    sums[0] += pages_of(q.to, st.page_shift) - q.fresh;
    sums[1] += q.count;
  }
#pragma unroll
  for (int k = 0; k < kFirst; ++k) sums[2] += __popc(early[k]);
  for (int w = w0 + kFirst; w < w1; ++w) sums[2] += __popc(word(w));
  block_scan<4>(sums, before, total, l.part + kWaves);
  int64_t offset = before[0], start = before[1];
  const int64_t n_take = total[0];
  const bool possible = total[3] == 0 && total[1] <= a.n_tokens, done = possible && n_take <= total[2];
  if (t == 0 && a.n == 0) a.starts[0] = 0;
  if (t == 0) *a.missing = possible ? (int32_t)max((int64_t)0, n_take - total[2]) : -1;

  for (int i = r0; i < r1; ++i) {
    Request q = get(i);
    if (!done) {
      q.to = q.from, q.count = 0, q.last = -1, q.fresh = pages_of(q.from, st.page_shift);
      offset = start = 0;
    }
    q.offset = (int32_t)offset, q.start = (int32_t)start;
    offset += pages_of(q.to, st.page_shift) - q.fresh;
    start += q.count;
    a.requests[i] = q;
    a.starts[i] = q.start;
    if (i == a.n - 1) a.starts[a.n] = (int32_t)start;
    a.step_lens[i] = q.to;
    if (q.seq >= 0 && q.count) st.lens[q.seq] = q.to;
    if (q.last >= 0) atomicSub(&st.refs[q.last], 1);
  }
  if (!done || n_take == 0) return;
  if (words <= kBases) {
    // a wave takes two words at a time, a lane a page
    int64_t rank = before[2];
#pragma unroll
    for (int k = 0; k < kFirst; ++k) {
      if (w0 + k < w1) l.bases[w0 + k] = (int32_t)rank;
      rank += __popc(early[k]);
    }
    for (int w = w0 + kFirst; w < w1; ++w) l.bases[w] = (int32_t)rank, rank += __popc(word(w));
    __syncthreads();
    const int lane = t & 63, b = lane & 31;
    for (int w2 = t >> 6 << 1; w2 < words && l.bases[w2] < n_take; w2 += 2 * kWaves) {
      const int w = w2 + (lane >> 5);
      const uint32_t x = w < words ? word(w) : 0;
      const int r = l.bases[min(w, words - 1)] + __popc(x & ((1u << b) - 1));
      const bool taken = (x >> b & 1) && r < n_take;
      if (taken) a.list[r] = 32 * w + b, st.refs[32 * w + b] = 1;
      const uint64_t both = __ballot(taken);
      const uint32_t gone = lane < 32 ? (uint32_t)both : (uint32_t)(both >> 32);
      if (b == 0 && gone) st.free[w] &= ~gone;
    }
    return;
  }
  int64_t rank = before[2];
  for (int w = w0; w < w1 && rank < n_take; ++w) {
    const uint32_t x = word(w);
    uint32_t left = x;
    for (; left && rank < n_take; ++rank) {
      const int b = __builtin_ctz(left);
      left &= left - 1;
      a.list[rank] = 32 * w + b;
      st.refs[32 * w + b] = 1;
    }
    if (left != x) st.free[w] &= ~(x ^ left);
  }
}

// What follows for one request, from thread `t` of `threads`: its table, its
// new entries and its tokens' places. Only entries that the request gets new
// are written to the tables, and none of those are read. The three calls above:
// 3.0, 4.0 and 6.1 us (6 MB).
__device__ void emit(const Extend& a, int i, int t, int threads) {
  const PageState& st = a.state;
  const Request q = a.requests[i];
  const int have = q.fresh, need = pages_of(q.to, st.page_shift);
  int32_t* const row = st.tables + (int64_t)max(q.seq, 0) * st.width;
  constexpr int kLoads = 8;  // on their way at once
  for (int j0 = t; j0 < a.width; j0 += threads * kLoads) {
    int32_t p[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int j = j0 + k * threads;
      p[k] = -1;
      if (j < min(need, a.width)) p[k] = j < have ? row[j] : a.list[q.offset + j - have];
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int j = j0 + k * threads;
      if (j >= a.width) break;
      if (j >= have && j < need) row[j] = p[k];
      a.step_tables[(int64_t)i * a.width + j] = p[k];
    }
  }
  if (t == 0) a.src[i] = q.last, a.dst[i] = q.last >= 0 ? a.list[q.offset] : -1;
  for (int j = t; j < q.count; j += threads) {
    const int at = q.from + j, place = at >> st.page_shift;
    const int32_t p = place < have ? row[place] : a.list[q.offset + place - have];
    a.positions[q.start + j] = at;
    a.slots[q.start + j] = p >= 0 && p < st.pages ? ((int64_t)p << st.page_shift) + (at & ((1 << st.page_shift) - 1)) : -1;
  }
}

// Places of the outputs behind the last token: position 0, no slot.
__device__ void pad(const Extend& a, int t, int threads) {
  for (int64_t j = a.starts[a.n] + t; j < a.n_tokens; j += threads) a.positions[j] = 0, a.slots[j] = -1;
}

template <bool ALL, bool ONE>
__global__ __launch_bounds__(kThreads) void plan_kernel(Extend a) {
  extern __shared__ uint32_t seen[];
  __shared__ PlanLds l;
  plan<ONE>(a, seen, l);
  if (!ALL) return;
  __syncthreads();
  for (int i = threadIdx.x >> 6; i < a.n; i += kWaves) emit(a, i, threadIdx.x & 63, 64);
  pad(a, threadIdx.x, kThreads);
}

__global__ __launch_bounds__(kRowThreads) void emit_kernel(Extend a) {
  const int t = blockIdx.y * kRowThreads + threadIdx.x, threads = gridDim.y * kRowThreads;
  if ((int)blockIdx.x < a.n) emit(a, blockIdx.x, t, threads);
  else pad(a, t, threads);
}

// A work-group cuts a sequence. 48 that lose a token 3.0 us, 256 with shared
// pages 6.6, 700 whole prompts 4.7 (13 with an atomic operation for every page
// and bit): bound by the chain of reads from a length to a page's owners.
__global__ __launch_bounds__(kRowThreads) void truncate_kernel(PageState st, const int32_t* seqs, const int32_t* to, int n) {
  const int i = blockIdx.x;
  const int32_t seq = seqs[i];
  if (seq < 0 || seq >= st.sequences) return;
  bool twice = false;  // only the first of several cuts counts
  for (int j = threadIdx.x; j < i; j += kRowThreads) twice |= seqs[j] == seq;
  const int32_t from = min((int64_t)max(st.lens[seq], 0), (int64_t)st.width << st.page_shift);
  const int32_t keep = to[i];
  if (__syncthreads_or(twice) || keep < 0 || keep >= from) return;
  const int p0 = pages_of(keep, st.page_shift), p1 = pages_of(from, st.page_shift);
  int32_t* const row = st.tables + (int64_t)seq * st.width;
  for (int j0 = p0; j0 < p1; j0 += kRowThreads) {
    const int j = j0 + threadIdx.x;
    int32_t p = -1;
    if (j < p1) p = row[j], row[j] = -1;
    bool freed = false;
    if (p >= 0 && p < st.pages) {
      // a page of one owner is nobody else's to count
      if (st.refs[p] == 1) st.refs[p] = 0, freed = true;
      else freed = atomicSub(&st.refs[p], 1) == 1;
    }
    // its bit, with those of the wave's other pages in the same word
    for (uint64_t left = __ballot(freed); left;) {
      const int w = __builtin_amdgcn_readlane(p, __builtin_ctzll(left)) >> 5;
      const bool here = freed && p >> 5 == w;
      uint32_t bits = here ? 1u << (p & 31) : 0;
#pragma unroll
      for (int d = 32; d; d >>= 1) bits |= __shfl_xor(bits, d, 64);
      if (threadIdx.x % 64 == 0) atomicOr(&st.free[w], bits);
      left &= ~__ballot(here);
    }
  }
  if (threadIdx.x == 0) st.lens[seq] = keep;
}

// A work-group makes a fork: 192 in 4.1 us.
__global__ __launch_bounds__(kRowThreads) void fork_kernel(PageState st, const int32_t* seqs, const int32_t* into, int n) {
  const int i = blockIdx.x;
  const int32_t from = seqs[i], to = into[i];
  if (from < 0 || from >= st.sequences || to < 0 || to >= st.sequences) return;
  bool clash = false;  // what another pair names to be written is neither read nor written
  for (int j = threadIdx.x; j < n; j += kRowThreads) {
    const bool other = into[j] >= 0 && into[j] < st.sequences && seqs[j] >= 0 && seqs[j] < st.sequences;
    clash |= seqs[j] == to || (other && (into[j] == from || (j < i && into[j] == to)));
  }
  const int32_t len = min((int64_t)max(st.lens[from], 0), (int64_t)st.width << st.page_shift);
  const bool taken = st.lens[to] != 0;
  if (__syncthreads_or(clash) || taken) return;
  const int pages = pages_of(len, st.page_shift);
  const int32_t* const row = st.tables + (int64_t)from * st.width;
  int32_t* const out = st.tables + (int64_t)to * st.width;
  for (int j = threadIdx.x; j < pages; j += kRowThreads) {
    const int32_t p = row[j];
    out[j] = p;
    if (p >= 0 && p < st.pages) atomicAdd(&st.refs[p], 1);
  }
  if (threadIdx.x == 0) st.lens[to] = len;
}

// ---- neighbours with the same first pages ----

struct Prefixes {
  const int32_t* tables;
  int64_t stride;
  int width;
  const int32_t* lens;
  int n, page_shift;
  int64_t least;
  int32_t *groups, *shared, *runs;
};

// One wave: the first pages that sequence b and the one before it both have whole.
__device__ int common_pages(const Prefixes& a, int b) {
  const int lane = threadIdx.x & 63;
  const int whole = min(min(max(a.lens[b], 0), max(a.lens[b - 1], 0)) >> a.page_shift, a.width);
  const int32_t* const x = a.tables + (b - 1) * a.stride;
  const int32_t* const y = a.tables + b * a.stride;
  constexpr int kLoads = 8;
  for (int j0 = 0; j0 < whole; j0 += 64 * kLoads) {
    bool differ[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int j = j0 + 64 * k + lane;
      differ[k] = j < whole && x[j] != y[j];
    }
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const uint64_t m = __ballot(differ[k]);
      if (m) return j0 + 64 * k + __builtin_ctzll(m);
    }
  }
  return whole;
}

__device__ __forceinline__ void find_run(const Prefixes& a, int b) {
  const int run = b ? common_pages(a, b) : 0;
  if ((threadIdx.x & 63) == 0) a.runs[b] = ((int64_t)run << a.page_shift) >= a.least && run ? run << a.page_shift : 0;
}

__device__ void group_runs(const Prefixes& a, int64_t* part) {
  const int t = threadIdx.x, lane = t & 63, run = (a.n + kThreads - 1) / kThreads, b0 = min(t * run, a.n), b1 = min(b0 + run, a.n);
  int64_t begun[1] = {0}, first[1], all[1];
  for (int b = b0; b < b1; ++b) begun[0] += a.runs[b] == 0;
  block_scan<1>(begun, first, all, part);
  int g = (int)first[0];
  const int total = (int)all[0];
  for (int b = b0; b < b1; ++b)
    if (a.runs[b] == 0) a.groups[g++] = b;
  for (int i = total + t; i <= a.n; i += kThreads) a.groups[i] = a.n;
  __syncthreads();
  // the least of a group's runs: a lane has a group, those of many sequences are gone through by all lanes
  constexpr int kFew = 8;
  for (int g0 = t - lane; g0 < a.n; g0 += kThreads) {
    const int i = g0 + lane;
    const int first = i < total ? a.groups[i] : 0, end = i < total ? a.groups[i + 1] : 0;
    int least = 0;
    if (end - first > 1 && end - first <= kFew) {
      least = 0x7FFFFFFF;
      for (int b = first + 1; b < end; ++b) least = min(least, a.runs[b]);
    }
    for (uint64_t many = __ballot(end - first > kFew); many; many &= many - 1) {
      const int of = __builtin_ctzll(many), f = __builtin_amdgcn_readlane(first, of), e = __builtin_amdgcn_readlane(end, of);
      int m = 0x7FFFFFFF;
      for (int b = f + 1 + lane; b < e; b += 64) m = min(m, a.runs[b]);
#pragma unroll
      for (int d = 32; d; d >>= 1) m = min(m, __shfl_xor(m, d, 64));
      if (lane == of) least = m;
    }
    if (i < a.n) a.shared[i] = least;
  }
}

template <bool ALL>
__global__ __launch_bounds__(kThreads) void group_kernel(Prefixes a) {
  __shared__ int64_t part[kWaves];
  if (ALL) {
    for (int b = threadIdx.x >> 6; b < a.n; b += kWaves) find_run(a, b);
    __syncthreads();
  }
  group_runs(a, part);
}

__global__ __launch_bounds__(64) void run_kernel(Prefixes a) { find_run(a, blockIdx.x); }

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

void check_count(int64_t n, const char* what) {
  if (n < 0 || n > 65535) throw std::invalid_argument(std::string(what) + " must be 0 to 65535");
}

}  // namespace

int64_t extend_workspace(int64_t n, int64_t pages) {
  return round16(n * (int64_t)sizeof(Request)) + round16(4 * pages) + round16(4 * n);
}

void extend_tables(const PageState& state, const ExtendArgs& a, hipStream_t s) {
  check_count(a.n, "requests");
  if (state.sequences > kSequences) throw std::invalid_argument("the sequences are too many (too large)");
  if (a.n_tokens > 0x7FFFFFFF) throw std::invalid_argument("n_tokens is too large");
  const int64_t bytes = extend_workspace(a.n, state.pages);
  if (a.workspace_bytes < bytes || !a.workspace || ((uintptr_t)a.workspace & 15u))
    throw std::invalid_argument("workspace must be 16-byte aligned and hold " + std::to_string(bytes) + " bytes");
  Extend p{};
  p.state = state, p.seqs = a.seqs, p.counts = a.counts, p.n = (int)a.n, p.width = a.width, p.n_tokens = a.n_tokens;
  p.positions = a.positions, p.slots = a.slots, p.starts = a.starts;
  p.step_tables = a.step_tables, p.step_lens = a.step_lens, p.src = a.src, p.dst = a.dst, p.missing = a.missing;
  char* const w = (char*)a.workspace;
  p.requests = (Request*)w;
  p.list = (int32_t*)(w + round16(a.n * (int64_t)sizeof(Request)));
  p.growers = (int32_t*)((char*)p.list + round16(4 * (int64_t)state.pages));
  const size_t lds = ((size_t)state.sequences + 31) / 32 * 4;
  // What little there is to write is written by the planning work-group's 16 waves,
  // a request each: a second kernel is a launch. Next tokens with the truncation back,
  // in a graph (and launched one by one), one kernel / two: 16 requests with tables of
  // 40 10.9 / 11.5 us (12.5 / 14.9), of 256 11.2 / 11.4 (13.3 / 15.3); 32 with tables
  // of 40 12.4 / 11.5 (12.4 / 15.0); 64 of 8 15.3 / 12.2 (15.9 / 14.9), 48 of 600
  // 16.6 / 11.9; 4 with tables of 250 and 1,000 tokens each 14.1 / 12.8.
  const bool all = a.n <= 2 * kWaves && a.n * a.width + a.n_tokens <= 512 * std::max<int64_t>(1, a.n);
  const bool one = a.n <= kThreads;
  auto kernel = all ? plan_kernel<true, true> : one ? plan_kernel<false, true> : plan_kernel<false, false>;
  if (lds > 8192)  // with what the kernel has anyway more than 64 KB
    hip_check(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "extend tables");
  kernel<<<1, kThreads, lds, s>>>(p);
  hip_check(hipGetLastError(), "extend tables");
  if (all) return;
  const int64_t each = std::max<int64_t>((a.n_tokens + a.n) / (a.n + 1), a.width);
  const dim3 grid((unsigned)a.n + 1, (unsigned)std::clamp<int64_t>(each / (8 * kRowThreads), 1, 64));
  emit_kernel<<<grid, kRowThreads, 0, s>>>(p);
  hip_check(hipGetLastError(), "extend tables");
}

void truncate_tables(const PageState& state, const int32_t* seqs, const int32_t* to, int64_t n, hipStream_t s) {
  check_count(n, "requests");
  if (n == 0) return;
  truncate_kernel<<<(unsigned)n, kRowThreads, 0, s>>>(state, seqs, to, (int)n);
  hip_check(hipGetLastError(), "truncate tables");
}

void fork_tables(const PageState& state, const int32_t* seqs, const int32_t* into, int64_t n, hipStream_t s) {
  check_count(n, "requests");
  if (n == 0) return;
  fork_kernel<<<(unsigned)n, kRowThreads, 0, s>>>(state, seqs, into, (int)n);
  hip_check(hipGetLastError(), "fork tables");
}

int64_t prefixes_workspace(int64_t batch) { return round16(4 * batch); }

void shared_prefixes(const int32_t* tables, int64_t stride, int64_t width, const int32_t* lens, int64_t batch,
                     int32_t page_shift, int64_t least, int32_t* groups, int32_t* shared, void* workspace,
                     int64_t workspace_bytes, hipStream_t s) {
  check_count(batch, "batch");
  if (workspace_bytes < prefixes_workspace(batch) || (batch && !workspace))
    throw std::invalid_argument("workspace must hold " + std::to_string(prefixes_workspace(batch)) + " bytes");
  Prefixes p{tables, stride, (int)width, lens, (int)batch, page_shift, least, groups, shared, (int32_t*)workspace};
  // Few sequences' prefixes are found by the grouping work-group's waves: 16 with
  // tables of 64 4.1 us, 5.0 with a kernel before it, of 4,096 14.2 and 14.6; 32 of
  // 64 4.9 and 5.4, of 512 6.3 and 5.8; 48 of 64 5.9 and 5.3, 1,000 of 64 65 and 6.7.
  if (batch <= kWaves || (batch <= 2 * kWaves && batch * width <= 8192)) {
    group_kernel<true><<<1, kThreads, 0, s>>>(p);
  } else {
    run_kernel<<<(unsigned)batch, 64, 0, s>>>(p);
    hip_check(hipGetLastError(), "shared prefixes");
    group_kernel<false><<<1, kThreads, 0, s>>>(p);
  }
  hip_check(hipGetLastError(), "shared prefixes");
}

}  // namespace jasper_amd
