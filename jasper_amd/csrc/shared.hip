// shared.hip -- attention of one new token per sequence where groups of
// sequences begin with the same tokens, which are read once for all of them.
//
// With n sequences of a group and gh query heads to a key head, the scores of
// the group's first S tokens are one product of M = n gh query rows with S key
// rows, and softmax statistics put what a row saw of them together with what it
// saw of its own tokens: out = sum_i 2^(ref_i - ref) o_i / sum_i 2^(ref_i -
// ref) sum_i over the parts i. So the work is streams of tokens under some
// query rows, shared out evenly over the work-groups:
//  wide  a group's prefix under more than 16 rows: a work-group takes tiles of
//        tokens into LDS, its waves 32 rows each (or the same rows and other
//        tokens of the tile), on 32x32x16 products;
//  thin  a group's prefix under up to 16 rows, and
//  own   what a sequence reads by itself: a wave each, past LDS (attend.hpp).
// A second kernel joins the parts of every row.
#include "kvcache.hpp"

#include "attend.hpp"
#include "graph.hpp"
#include "kvtypes.hpp"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace jasper_amd {

namespace {

using namespace attention;

constexpr int kBatch = 512;      // sequences of a launch
constexpr int kGroups = 256;     // work-groups: one for each compute unit
constexpr int kStage = 512;      // row offsets of a wave, in LDS
constexpr int kJoin = 256;       // threads of a joining work-group
constexpr int kPages = 1024;     // of a wide stream's table, in LDS
constexpr int kTeam = 8;         // work-groups of a team at most
// What beginning a wide stream and a tile of it cost a work-group, in tiles of 32
// tokens of a wave: it waits for pages, queries and tiles, and its waves join.
// 64 sequences over 16,384 tokens, 64 in four groups over 8,000: 66.4 and 53.4
// us; with tiles of 2 71.6 and 54.9, of 1 and a start of 6 81.4 and 59.6. Tiles of
// heads of 256 values have half the tokens: 32 over 32,768 97.1, with 3 99.0.
constexpr int kWideStart = 14;
constexpr int wide_tile(int dt) { return dt == 256 ? 2 : 3; }
constexpr int kLeast = 2;      // tiles of a wave

constexpr int waves_of(int dt) { return dt == 256 ? 4 : 8; }    // of a work-group
constexpr int tokens_of(int dt) { return 8192 / dt; }             // of a wide tile: 16 KB of K
constexpr int kRows = 128;       // query rows of a work-group
__host__ __device__ constexpr int part_row(int dt) { return dt + 4; }  // floats: sums of V, ref, sum

struct Shared {
  Params a;  // lists: the key heads
  const int32_t *groups, *shared;
  int n_groups;
  bool far;  // rows of a page are more than 2^31 bytes apart
  int first, count;  // sequences of this launch
  int4* prefix_ends;  // [count * q_heads]: the work-group that begins the prefix, how many have parts, the row in them, the step from one to the next (0: they are waves)
  int2* own_ends;     // [count * q_heads]: the wave that begins what a sequence has itself, how many have parts
  float *prefix_first, *own_first;  // [count * q_heads] part rows: the parts that begin a stream
  float *wide_rest;   // [work-groups][rows of a wide tile]: parts that go on with one
  float *wave_rest;   // [waves][16]
};

// What every work-group finds out for itself, in LDS. Of group members only the
// first and last that have the whole prefix count, as leader and last, at the
// place of the group's first sequence. wide, thin, own: units before.
struct Layout {
  int from[kBatch];  // tokens that a sequence leaves to its group
  int leader[kBatch], last[kBatch];
  int wide[kBatch], thin[kBatch], own[kBatch];
  int len[kBatch];
  // a group that began in an earlier launch: where, its prefix, and its first
  // sequence that is long enough (none: kNone)
  int cut_begin, cut_shared, cut;
  int longest[8];  // tiles of the longest stream that is not wide, by waves
  int wider;  // whether a group has more rows than a work-group
  int totals[3];
  int part[3][8];
};

constexpr int kNone = 0x7FFFFFFF;

__device__ __forceinline__ int length_of(const Shared& p, int i) { return min(max(p.a.lens[p.first + i], 0), p.a.limit); }

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Whether sequences read a prefix at place i: two or more, or what is left of a cut group.
__device__ __forceinline__ bool shares(const Layout& l, int i) {
  return l.leader[i] < l.last[i] || (i == 0 && l.cut != kNone && l.last[0] >= 0);
}

// The sequence in whose table it is.
__device__ __forceinline__ int source_of(const Shared& p, const Layout& l, int i) {
  return i == 0 && l.cut != kNone ? l.cut : p.first + l.leader[i];
}

// The sum of x over the lanes up to this one, without LDS.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // rows of 16 lanes, shifted by 1, 2, 4 and 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // lane 15 of a row to the next one
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // lane 31 to the last two
  return x;
}

// In lane 63: the largest x of a wave, none below 0.
__device__ __forceinline__ int wave_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));
  return x;
}

// For three numbers at once: their sums over the threads before, and over all.
template <int NW>
__device__ __forceinline__ void block_scan(const int (&x)[3], int (&before)[3], int (&total)[3], int (&part)[3][8]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    incl[k] = wave_scan(x[k]);
    if (lane == 63) part[k][wave] = incl[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    before[k] = incl[k] - x[k], total[k] = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w == wave) before[k] += total[k];
      total[k] += part[k][w];
    }
  }
}

// The row tiles of a wide group, as blocks of a team.
__device__ __forceinline__ int blocks_of(int rows, int team) { return ceil_div(ceil_div(rows, kRows), team); }

// Work-groups form teams: those of one take the same tokens under different
// rows, on one XCD, so that its L2 reads them from memory once (512 rows over
// 131,072 tokens of 8 heads: 426 us, 446 without). Groups
// of unlike size might leave members without rows; where that would be more than a
// quarter more tiles there are no teams (512 rows over 131,072 tokens beside 128 over
// 32,768, 1.18 times the tiles: 480 us with teams, 498 without; over 65,536, 1.33
// times: 540 and 509; 512 and 384 over 16,384, 1.14 times: 127 and 125).
// Returns the work-groups of a team.
template <int NW, int DT>
__device__ int lay_out(const Shared& p, Layout& l) {
  constexpr int kThreads = NW * 64, kRun = kBatch / kThreads, TT = tokens_of(DT);
  const int t = threadIdx.x, gh = p.a.group;
  for (int i = t; i < kBatch; i += kThreads) l.leader[i] = kNone, l.last[i] = -1, l.from[i] = 0, l.own[i] = 0;
  if (t == 0) l.cut_begin = p.first, l.cut_shared = 0, l.cut = kNone, l.wider = 0;
  // the groups' first sequences and prefixes, where there is room for them
  const bool held = p.n_groups <= kBatch;
  if (held)
    for (int i = t; i < p.n_groups; i += kThreads) l.wide[i] = p.groups[i], l.thin[i] = p.shared[i];
  const int end = p.groups[p.n_groups];
  __syncthreads();
  for (int i = t; i < p.count; i += kThreads) {
    const int b = p.first + i, len = length_of(p, i);
    l.len[i] = len;
    int lo = 0, hi = p.n_groups;  // the last group that begins at or before b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if ((held ? l.wide[mid] : p.groups[mid]) <= b) lo = mid + 1;
      else hi = mid;
    }
    const int g = lo - 1;
    if (g < 0 || b >= end) continue;
    const int shared = held ? l.thin[g] : p.shared[g], begin = held ? l.wide[g] : p.groups[g], slot = max(begin, p.first) - p.first;
    if (i == 0) l.cut_begin = max(begin, 0), l.cut_shared = shared;
    if (shared <= 0 || len < shared) continue;
    l.from[i] = shared, l.own[i] = slot;
    atomicMin(&l.leader[slot], i);
    atomicMax(&l.last[slot], i);
  }
  __syncthreads();
  if (p.first) {
    for (int b = l.cut_begin + t; b < p.first; b += kThreads)
      if (l.cut_shared > 0 && length_of(p, b - p.first) >= l.cut_shared) atomicMin(&l.cut, b);
    __syncthreads();
  }
  const auto rows_of = [&](int i) { return shares(l, i) ? (l.last[i] - l.leader[i] + 1) * gh : 0; };
  // the team that the largest group would have, and what all groups would make of it
  int most = 0, team = 1;
  for (int i = t; i < p.count; i += kThreads) most = max(most, ceil_div(rows_of(i), kRows));
  if (most > 1) l.wider = 1;
  __syncthreads();
  if (l.wider) {
#pragma unroll
    for (int d = 32; d; d >>= 1) most = max(most, __shfl_xor(most, d, 64));
    if ((t & 63) == 0) l.part[0][t >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) most = max(most, l.part[0][w]);
    __syncthreads();
    team = min(ceil_div(most, ceil_div(most, kTeam)), (int)(gridDim.x % 8 ? gridDim.x : gridDim.x / 8));
    int used[3] = {0, 0, 0}, unused[3], all[3];
    for (int i = t; i < p.count; i += kThreads) {
      const int rows = rows_of(i);
      if (rows <= kHeads) continue;
      const int tiles = ceil_div(l.from[l.leader[i]], TT);
      used[0] += ceil_div(rows, kRows) * tiles, used[1] += blocks_of(rows, team) * team * tiles;
    }
    block_scan<NW>(used, unused, all, l.part);
    if (all[1] > all[0] + all[0] / 4) team = 1;
    __syncthreads();
  }
  const int tile_cost = wide_tile(DT) * team, start_cost = kWideStart * team;
  int units[3] = {0, 0, 0}, before[3], total[3];
  int each[3][kRun], longest = 0;
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = t * kRun + k;
    each[0][k] = units[0], each[1][k] = units[1], each[2][k] = units[2];
    if (i >= p.count) continue;
    const int rows = rows_of(i);
    if (rows) {
      const int shared = l.from[l.leader[i]];
      if (rows > kHeads) units[0] += p.a.heads * blocks_of(rows, team) * (start_cost + ceil_div(shared, TT) * tile_cost);
      else units[1] += p.a.heads * (kStart + ceil_div(shared, kTile)), longest = max(longest, ceil_div(shared, kTile));
    }
    const int slot = l.own[i], from = shares(l, slot) ? l.from[i] : 0;
    const int tiles = max(1, ceil_div(l.len[i] - (from & ~7), kTile));
    units[2] += p.a.heads * p.a.head_tiles * (kStart + tiles), longest = max(longest, tiles);
  }
  longest = wave_max(longest);
  if ((t & 63) == 63) l.longest[t >> 6] = longest;
  block_scan<NW>(units, before, total, l.part);
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = t * kRun + k, slot = l.own[i];
    if (!shares(l, slot)) l.from[i] = 0;  // alone with its prefix; nobody else reads this place
    l.wide[i] = before[0] + each[0][k], l.thin[i] = before[1] + each[1][k], l.own[i] = before[2] + each[2][k];
  }
  if (t == 0) l.totals[0] = total[0], l.totals[1] = total[1], l.totals[2] = total[2];
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(team);
}

// The last i with at[i] <= u, of n <= kBatch; for a whole wave.
__device__ __forceinline__ int find(const int* at, int n, int u) {
  constexpr int kRun = kBatch / 64;
  const int lane = threadIdx.x & 63;
  const int run = __popcll(__ballot(lane * kRun < n && at[lane * kRun] <= u)) - 1;
  const int i = run * kRun + lane;
  return run * kRun + __popcll(__ballot(lane < kRun && i < n && at[i] <= u)) - 1;
}

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ floatx16 mfma32(Frag a, Frag b, floatx16 c) {
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
  if constexpr (std::is_same_v<T, f16>)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
}

// Lane i of 16 gives the address of four values in row i / 4 of a 4 x 16 block
// of LDS, its columns 4 (i % 4) on, and gets column i.
__device__ __forceinline__ uintx2 read_column(const char* p) {
  return __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                        (__attribute__((address_space(3))) shortx4*)(uintptr_t)(p)));
}

// A stretch of a wide stream.
struct WidePart {
  int leader;  // the group's first sequence here, counted from the launch's
  int source;  // the sequence whose table has the prefix
  int head, row0, rows, tokens;
  int c, c1;  // its tiles
};

// Where a stretch ends that begins with tile c of `tokens` tokens: before c1, and
// with the last of kPages pages, of which the first may have begun before the tile.
__host__ __device__ constexpr int stretch_end(int c, int c1, int tokens, int page_shift) {
  const int64_t last = ((int64_t)c * tokens >> page_shift) + kPages;
  const int64_t end = (last << page_shift) / tokens;
  return end < c1 ? (int)end : c1;
}

constexpr bool stretches_fit() {
  for (int tokens = tokens_of(256); tokens <= tokens_of(64); tokens *= 2)
    for (int shift = 3; shift <= 8; ++shift)
      for (int c = 0, far = (int)(0x7FFFFF00ll / tokens); c < 32; ++c)
        for (const int from : {c, far - 40'000 + c, far - c - 1}) {
          const int end = stretch_end(from, far, tokens, shift);
          const int64_t first = (int64_t)from * tokens >> shift, last = ((int64_t)end * tokens - 1) >> shift;
          if (end <= from || last - first >= kPages) return false;
          if (end < far && ((((int64_t)end + 1) * tokens - 1) >> shift) - first < kPages) return false;  // there was room
        }
  return true;
}
static_assert(stretches_fit(), "a stretch has at least a tile and at most kPages pages");

// A wave's 64 times 16 bytes from memory to LDS at `to` on, in the lanes' order,
// past the registers; lanes that do not take part leave theirs out. They arrive
// in order and are waited for by loads_left. (The compiler does not see these
// writes to LDS coming: they go to tiles that nobody reads before a barrier.)
// Nor does it see the instruction's own hazards: one wait state after m0 is
// written, five from a vector instruction that writes the scalar base
// (readfirstlane) on, of which the write of m0 is one. It is told of m0, which it
// reserves and warns of: nothing is kept there.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds(const void* from, uint32_t to) {
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void load_lds(const char* base, uint32_t offset, uint32_t to) {
  const uint64_t at = (uint64_t)base;
  base = (const char*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at));
  to = __builtin_amdgcn_readfirstlane(to);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void loads_left() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// One work-group over tiles [c, c1) of a wide stream; the sums end up in the
// waves of the tile's first tokens. LDS holds four tiles of K and V: while the
// weights of one are found and multiplied with its values, the next one's scores
// are multiplied, and two more are on their way. Waves are four times 32 query
// rows, and as many for other tokens of the tile as there are more.
//
// S^T = K Q^T and O^T = V^T P^T on 32x32x16 products, hi = lane / 32. A lane's
// column is a query row all the way: S comes out with the scores of rows 8 a + 4
// hi + c of K in register 4 a + c, so the rows are put into LDS with bits 2 and
// 3 of the token exchanged, and registers 8 k on hold tokens 16 k + 8 hi on, as P
// has to be as the operand of the second product: nothing crosses lanes. V^T is
// read from V's rows by LDS reads that transpose. The 16-byte chunks of a row are
// exchanged by bits of the row so that lanes read from different banks: of reads
// of 16 bytes 16 lanes at once (8.6 cycles a read of a wave, 10.5 otherwise), of
// those that transpose 16 and 32 lanes (5.6 cycles, 8.1 without).
template <typename T, bool F8, int DT, bool FULL>
struct Wide {
  typedef std::conditional_t<F8, f16, T> PT;
  static constexpr int NW = waves_of(DT), TT = tokens_of(DT), TW = NW / 4, TPW = TT / TW, NB = TPW / 32;
  static constexpr int RB = DT * 2, CH = RB / 16;
  static constexpr int kThreads = NW * 64, kTileBytes = TT * RB, kBuffers = 4, kAhead = F8 ? 4 : 3;
  // 16-byte loads of a row; of a thread for a tile of K; rows of a wave's load
  static constexpr int UNITS = F8 ? CH / 2 : CH, ITER = TT * UNITS / kThreads, RPL = 64 / UNITS;
  static constexpr int KS = DT / 16, DB = DT / 32, ES = F8 ? 1 : 2;
  static constexpr float kLag = 3.f, kTop = std::is_same_v<PT, f16> ? 12.f : -kLag;  // as in attend_tiles
  static constexpr int kLds = kBuffers * 2 * kTileBytes;
  static_assert(NB >= 1 && ITER >= 1, "a tile is too small");
  static_assert((TW - 1) * 4 * (DB * 16 + 2) * 64 * 4 <= kLds, "the waves' sums do not fit");

  typedef floatx16 Scores[NB];
  struct Staged {
    uintx4 k[F8 ? ITER : 1], v[F8 ? ITER : 1];
  };

  const Shared& p;
  char* const lds;
  uint8_t (*const ok)[TT];
  int32_t* const held;     // kPages pages of the table, from page0 on
  int32_t* const masked;  // whether one of them is none, or rows are far apart
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave / TW, tw = wave % TW;

  Frag q[KS];
  floatx16 o[DB];
  float ref, use, sum, cs;
  bool holes;  // tokens without a page, or strides past 32 bits
  int32_t page_a[ITER], page_b[ITER];  // of a wave's loads: the pages of their first and second eight tokens
  uint32_t k_off[ITER], v_off[ITER];
  int page0;
  int tid, lane, hi;

  // What is worked out from a thread's index from here on is worked out from here
  // on: kept from further up in the kernel it would take most of the registers.
  __device__ __forceinline__ void place() {
    tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    lane = tid & 63, hi = lane >> 5;
  }

  __device__ char* k_tile(int b) const { return lds + b * 2 * kTileBytes; }
  __device__ char* v_tile(int b) const { return lds + b * 2 * kTileBytes + kTileBytes; }

  __device__ static __forceinline__ uint32_t lds_at(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
  }

  // The row of LDS that a thread's e-th 16 bytes are in, their place in it, and the token that is in a row.
  __device__ static __forceinline__ int row_of(int e, int t) { return (e * kThreads + t) / UNITS; }
  __device__ static __forceinline__ int slot_of(int e, int t) { return (e * kThreads + t) % UNITS; }
  __device__ static __forceinline__ int token_of(int m) { return (m & ~12) | (m & 4) << 1 | (m & 8) >> 1; }
  __device__ static __forceinline__ int k_key(int m) { return CH == 8 ? m >> 1 & 7 : m & 15; }
  __device__ static __forceinline__ int v_key(int m) { return CH == 8 ? (m & 3) << 1 : (m & 3) << 1 | (m & 1) << 3; }

  // The chunk of a row in memory that a thread's e-th place has.
  __device__ static __forceinline__ int chunk_of(int e, int t, bool of_k) {
    const int m = row_of(e, t), slot = slot_of(e, t);
    return F8 ? slot : slot ^ (of_k ? k_key(m) : v_key(m));
  }

  __device__ __forceinline__ bool whole(const WidePart& w, int tile) const { return !holes && (tile + 1) * TT <= w.tokens; }

  // The pages of a tile's tokens, from LDS (scalar loads from the table itself
  // would wait for memory every few tiles, and LDS reads with them).
  __device__ __forceinline__ void look(const WidePart& w, int tile) {
    const int last = w.tokens - 1;
#pragma unroll
    for (int e = 0; e < ITER; ++e) {
      const int m = (e * NW + wave) * RPL;  // the first row of the wave's load
      const int t = tile * TT + (RPL >= 8 ? m & ~15 : token_of(m) & ~7);
      page_a[e] = held[(min(t, last) >> p.a.page_shift) - page0];
      if constexpr (RPL >= 8) page_b[e] = held[(min(t + 8, last) >> p.a.page_shift) - page0];
    }
  }

  // Sends for a tile whose pages are known: to buffer b, or (e4m3, which is
  // widened on the way) to registers. This for a whole tile, and PART of 4 of it, as
  // the loads of all waves at once would stand in each other's way: a wave's four
  // took 500 to 790 of a step's 3000 cycles.
  template <int PART>
  __device__ __forceinline__ void fetch_part(const WidePart& w, int tile, int b, Staged& st) {
    const Params& a = p.a;
    const int64_t at = w.head * a.head_stride + (int64_t)(tile * TT & ((1 << a.page_shift) - 1)) * a.row_stride;
#pragma unroll
    for (int j = PART * 2 * ITER / 4; j < (PART + 1) * 2 * ITER / 4; ++j) {
      const int e = j / 2;
      const bool of_k = j % 2 == 0;
      const char* const base = of_k ? a.k : a.v;
      const int32_t pa = __builtin_amdgcn_readfirstlane(page_a[e]);
      const uint32_t off = of_k || F8 ? k_off[e] : v_off[e];
      const bool mine = FULL || chunk_of(e, tid, of_k) * (16 / ES) < a.dim;
      const char* from = base + (pa * a.page_stride + at) * ES;
      if constexpr (RPL >= 8) {
        const int32_t pb = __builtin_amdgcn_readfirstlane(page_b[e]);
        from = row_of(e, tid) & 4 ? base + (pb * a.page_stride + at) * ES : from;
      }
      if constexpr (F8) {
        uintx4& staged = of_k ? st.k[e] : st.v[e];
        if constexpr (!FULL) staged = uintx4{0, 0, 0, 0};
        if (mine) staged = *(const uintx4*)(from + off);
      } else {
        const uint32_t to = lds_at(of_k ? k_tile(b) : v_tile(b)) + (e * kThreads + wave * 64) * 16;
        if constexpr (RPL < 8) {
          if (mine) load_lds(from, off, to);
        } else {
          if (mine) load_lds(from + off, to);
        }
      }
    }
  }

  // The same for any tile, all of it. What is not there is zero, and not ok.
  __device__ __forceinline__ void fetch(const WidePart& w, int tile, int b, Staged& st) {
    if (whole(w, tile)) {
      fetch_part<0>(w, tile, b, st), fetch_part<1>(w, tile, b, st);
      fetch_part<2>(w, tile, b, st), fetch_part<3>(w, tile, b, st);
      return;
    }
    const Params& a = p.a;
    const int64_t at = w.head * a.head_stride + (int64_t)(tile * TT & ((1 << a.page_shift) - 1)) * a.row_stride;
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // this is rare: not worth registers through every step
#pragma unroll
    for (int e = 0; e < ITER; ++e) {
      const int m = row_of(e, thread), r = token_of(m), place = (e * kThreads + thread) * 16;
      const int32_t page = RPL >= 8 && m & 4 ? page_b[e] : page_a[e];
      const bool in = page >= 0 && page < a.pages && tile * TT + r < w.tokens;
      const int64_t row = (page * a.page_stride + at + (int64_t)(r & ((1 << a.page_shift) - 1)) * a.row_stride) * ES;
      const int kc = chunk_of(e, thread, true), vc = chunk_of(e, thread, false);
      const bool k_in = in && (FULL || kc * (16 / ES) < a.dim), v_in = in && (FULL || vc * (16 / ES) < a.dim);
      if constexpr (F8) {
        st.k[e] = st.v[e] = uintx4{0, 0, 0, 0};
        if (k_in) st.k[e] = *(const uintx4*)(a.k + row + kc * 16), st.v[e] = *(const uintx4*)(a.v + row + vc * 16);
      } else {
        const uint32_t run = (e * kThreads + wave * 64) * 16;
        if (k_in) load_lds(a.k + row + kc * 16, lds_at(k_tile(b)) + run);
        else *(uintx4*)(k_tile(b) + place) = uintx4{0, 0, 0, 0};
        if (v_in) load_lds(a.v + row + vc * 16, lds_at(v_tile(b)) + run);
        else *(uintx4*)(v_tile(b) + place) = uintx4{0, 0, 0, 0};
      }
      if (slot_of(e, thread) == 0) ok[b][m] = in;
    }
  }

  // e4m3: from the registers to buffer b.
  __device__ __forceinline__ void store(int b, const Staged& st) {
#pragma unroll
    for (int e = 0; e < ITER; ++e) {
      const int m = row_of(e, tid), slot = slot_of(e, tid);
      char* const kd = k_tile(b) + m * RB;
      char* const vd = v_tile(b) + m * RB;
      const uintx4 k = st.k[e], v = st.v[e];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t k0 = h ? k.z : k.x, k1 = h ? k.w : k.y, v0 = h ? v.z : v.x, v1 = h ? v.w : v.y;
        *(uintx4*)(kd + ((2 * slot + h) ^ k_key(m)) * 16) = uintx4{from_e4m3<T>(k0, false), from_e4m3<T>(k0, true), from_e4m3<T>(k1, false), from_e4m3<T>(k1, true)};
        *(uintx4*)(vd + ((2 * slot + h) ^ v_key(m)) * 16) = uintx4{from_e4m3<PT>(v0, false), from_e4m3<PT>(v0, true), from_e4m3<PT>(v1, false), from_e4m3<PT>(v1, true)};
      }
    }
  }

  // A wave's tokens of buffer b as operands of the first product.
  __device__ __forceinline__ void read_keys(int b, Frag (&f)[NB * KS]) const {
    const char* const kt = k_tile(b) + (tw * TPW + (lane & 31)) * RB;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < KS; ++e) f[n * KS + e] = *(const Frag*)(kt + n * 32 * RB + ((2 * e + hi) ^ k_key(lane & 31)) * 16);
  }

  __device__ __forceinline__ void scores(const Frag (&f)[NB * KS], Scores& s) const {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = 0;
#pragma unroll
      for (int e = 0; e < KS; ++e) s[n] = mfma32<T>(f[n * KS + e], q[e], s[n]);
    }
  }

  // Scores that are none left out; the reference moved where one is too large for it.
  __device__ __forceinline__ void settle(bool all, int b, Scores& s) {
    if (!all) {
      asm volatile("");  // a branch, not selects in every tile
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!ok[b][tw * TPW + n * 32 + 8 * (r / 4) + 4 * hi + r % 4]) s[n][r] = -__builtin_inff();
    }
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
    top *= cs;
    if (__any(top > ref + (kTop + kLag))) {
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float now = fmaxf(ref, top - kTop);
      const float to = now == -__builtin_inff() ? 0.f : now;
      const float keep = __builtin_amdgcn_exp2f(ref - to);
      sum *= keep;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= keep;
      ref = now, use = to;
    }
  }

  // The weights of scores in two terms of their type, as decode_attention's, so
  // that their rounding adds nothing to the output's own.
  __device__ __forceinline__ void weigh(const Scores& s, Frag (&hi)[NB * 2], Frag (&lo)[NB * 2]) {
#pragma unroll
    for (int n = 0; n < NB * 2; ++n)
#pragma unroll
      for (int r = 0; r < 8; r += 2) {
        const float y0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n / 2][n % 2 * 8 + r], cs, -use));
        const float y1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n / 2][n % 2 * 8 + r + 1], cs, -use));
        sum += y0 + y1;
        hi[n][r / 2] = pack2<PT>(y0, y1);
        const floatx2 back = unpack2<PT>(hi[n][r / 2]);
        lo[n][r / 2] = pack2<PT>(y0 - back.x, y1 - back.y);
      }
  }

  // Sixteen tokens, n * 16 on, of a wave's in buffer b as operands of the second product.
  __device__ __forceinline__ void read_values(int b, int n, Frag (&f)[DB]) const {
    // lane's place in the 4 x 16 blocks that it reads with 15 others
    const int i = lane & 15, g1 = lane >> 4 & 1;
    const char* const vt = v_tile(b) + (tw * TPW + n * 16 + 4 * hi + i / 4) * RB + 8 * (i & 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const char* const at = vt + ((4 * d + 2 * g1 + (i % 4) / 2) ^ v_key(i / 4)) * 16;
      const uintx2 v0 = read_column(at), v1 = read_column(at + 8 * RB);
      f[d] = Frag{v0.x, v0.y, v1.x, v1.y};
    }
  }

  __device__ __forceinline__ void add_values(const Frag (&f)[DB], Frag hi, Frag lo) {
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = mfma32<PT>(f[d], hi, o[d]);
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = mfma32<PT>(f[d], lo, o[d]);
  }

  __device__ __forceinline__ void values(int b, const Frag (&w)[NB * 2], const Frag (&lo)[NB * 2]) {
    Frag f[2][DB];
    read_values(b, 0, f[0]);
#pragma unroll
    for (int n = 0; n < NB * 2; ++n) {
      if (n + 1 < NB * 2) read_values(b, n + 1, f[n + 1 & 1]);
      __builtin_amdgcn_sched_barrier(0);
      add_values(f[n & 1], w[n], lo[n]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Tile t's values with tile t + 1's scores: what is on its way then is t + 2 and
  // t + 3. Reads of LDS go out well before their products and loads between
  // products; the compiler would put every read right before its product, and is
  // kept from it. Nothing here may spill: reading it back would wait for all loads.
  // STEADY: what is sent for is a whole tile. (To have the two waves of a SIMD take
  // turns, one with the vector units and one with the matrix cores, by barriers at
  // different places, gave nothing.)
  template <bool STEADY>
  __device__ __forceinline__ void step(const WidePart& w, int t, Scores& s, Staged& st) {
    const int b = t - w.c, to = (b + kAhead) & 3;
    Frag kf[NB * KS], wf[NB * 2], lf[NB * 2], vf[2][DB];
    const auto apart = [] { __builtin_amdgcn_sched_barrier(0); };
    const auto send = [&](auto part) {
      if constexpr (STEADY) fetch_part<decltype(part)::value>(w, t + kAhead, to, st);
      apart();
    };
    if constexpr (!F8) {
      if (STEADY || (t + 2 < w.c1 && whole(w, t + 2))) loads_left<2 * ITER>();
      else loads_left<0>();
    }
    __syncthreads();
    read_keys((b + 1) & 3, kf);
    apart();
    weigh(s, wf, lf);
    apart();
    if (F8 && t + 2 < w.c1) store((b + 2) & 3, st);
    if (!STEADY && t + kAhead < w.c1) fetch(w, t + kAhead, to, st);
    send(std::integral_constant<int, 0>{});
    read_values(b & 3, 0, vf[0]);
    apart();
    scores(kf, s);
    apart();
    send(std::integral_constant<int, 1>{});
#pragma unroll
    for (int n = 0; n < NB * 2; ++n) {
      if (n + 1 < NB * 2) read_values(b & 3, n + 1, vf[n + 1 & 1]);
      apart();
      add_values(vf[n & 1], wf[n], lf[n]);
      apart();
      if (n == 0) send(std::integral_constant<int, 2>{});
      if (n == 1) send(std::integral_constant<int, 3>{});
    }
    if (t + kAhead + 1 < w.c1) look(w, t + kAhead + 1);
    apart();
    settle(STEADY || whole(w, t + 1), (b + 1) & 3, s);
  }

  // A wave's part in a stretch whose first tiles are on their way.
  __device__ __forceinline__ void take(const WidePart& w, Staged (&st)[2]) {
    place();
    Scores s;
    {
      Frag kf[NB * KS];
      read_keys(0, kf);
      scores(kf, s);
    }
    settle(whole(w, w.c), 0, s);
    int t = w.c;
    const int steady = (holes ? 0 : min(w.c1, w.tokens / TT)) - kAhead;
    if constexpr (F8) {  // the registers take turns
      for (; t + 1 < steady; t += 2) {
        step<true>(w, t, s, st[0]);
        step<true>(w, t + 1, s, st[1]);
      }
      for (; t + 2 < w.c1; t += 2) {
        step<false>(w, t, s, st[0]);
        step<false>(w, t + 1, s, st[1]);
      }
      if (t + 1 < w.c1) step<false>(w, t, s, st[0]);
    } else {
      for (; t < steady; ++t) step<true>(w, t, s, st[0]);
      for (; t + 1 < w.c1; ++t) step<false>(w, t, s, st[0]);
    }
    Frag wf[NB * 2], lf[NB * 2];
    weigh(s, wf, lf);
    values((w.c1 - 1 - w.c) & 3, wf, lf);
  }

  __device__ __forceinline__ void run_stretch(const WidePart& w) {
    const Params& a = p.a;
    place();
    __syncthreads();  // what was in LDS before has been read
    if (tid == 0) *masked = p.far;
    page0 = w.c * TT >> a.page_shift;
    bool hole = false;
    const int n_pages = ((min(w.c1 * TT, w.tokens) - 1) >> a.page_shift) - page0 + 1;
    for (int i = tid; i < n_pages; i += kThreads) {
      const int32_t page = a.tables[w.source * a.table_stride + page0 + i];
      held[i] = page;
      hole = hole || page < 0 || page >= a.pages;
    }
    if (!FULL && !F8) {
#pragma unroll
      for (int e = 0; e < ITER; ++e)
        if (chunk_of(e, tid, true) * 8 >= a.dim)
          for (int b = 0; b < kBuffers; ++b) *(uintx4*)(k_tile(b) + (e * kThreads + tid) * 16) = uintx4{0, 0, 0, 0};
    }
    __syncthreads();
    if (hole) *masked = 1;
    look(w, w.c);
    __syncthreads();
    holes = __builtin_amdgcn_readfirstlane(*masked);
    Staged st[2];
    const int n = w.c1 - w.c;
    if constexpr (F8) {
      fetch(w, w.c, 0, st[0]);
      if (n > 1) look(w, w.c + 1), fetch(w, w.c + 1, 1, st[1]);
      store(0, st[0]);
      if (n > 2) look(w, w.c + 2), fetch(w, w.c + 2, 2, st[0]);
      if (n > 1) store(1, st[1]);
      if (n > 3) look(w, w.c + 3), fetch(w, w.c + 3, 3, st[1]);
      if (n > 4) look(w, w.c + 4);
    } else {
      for (int b = 0; b < min(n, 3); ++b) {
        if (b) look(w, w.c + b);
        fetch(w, w.c + b, b, st[0]);
      }
      if (n > 3) look(w, w.c + 3);
      if (n > 2 && whole(w, w.c + 2)) loads_left<4 * ITER>();
      else loads_left<0>();
    }
    __syncthreads();
    take(w, st);
  }

  __device__ void run(const WidePart& w) {
    const Params& a = p.a;
    place();
    const int row = rw * 32 + (lane & 31), at = w.row0 + row;
    const int member = w.leader + at / a.group, q_head = w.head * a.group + at % a.group;
    const char* const q_row = a.q + ((p.first + member) * a.q_stride + q_head * a.q_head) * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * hi;
      q[s] = Frag{0, 0, 0, 0};
      if (row < w.rows && (FULL || d < a.dim)) q[s] = *(const Frag*)(q_row + d * 2);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0;
    ref = -__builtin_inff(), use = 0.f, sum = 0.f;
    cs = a.scale * (a.k_scale ? a.k_scale[w.head] : 1.f);
    if (cs < 0.f) {  // the queries take the sign, so that the largest score is the largest product's
      cs = -cs;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] ^= 0x80008000u;
    }
    if (cs == 0.f) cs = 0x1p-126f;  // a masked score, -inf, times it stays that
#pragma unroll
    for (int e = 0; e < ITER; ++e) {
      const uint32_t r = (uint32_t)((token_of(row_of(e, tid)) & ((1 << a.page_shift) - 1)) * a.row_stride * ES);
      k_off[e] = r + chunk_of(e, tid, true) * 16, v_off[e] = r + chunk_of(e, tid, false) * 16;
    }
    // as many tiles as there is room for pages of, and again
    WidePart stretch = w;
    for (; stretch.c < w.c1; stretch.c = stretch.c1) {
      stretch.c1 = stretch_end(stretch.c, w.c1, TT, a.page_shift);
      run_stretch(stretch);
    }
    sum += __shfl_xor(sum, 32, 64);
    if constexpr (TW > 1) {
      // the waves of other tokens hand their sums over, 16 bytes of a lane at a time
      constexpr int kOne = (DB * 16 + 2) * 64;
      float* const all = (float*)lds;
      __syncthreads();
      if (tw) {
        float* const mine = all + ((tw - 1) * 4 + rw) * kOne;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4)
            *(floatx4*)(mine + ((d * 4 + r / 4) * 64 + lane) * 4) = floatx4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        *(floatx2*)(mine + DB * 16 * 64 + 2 * lane) = floatx2{ref, sum};
      }
      __syncthreads();
      if (tw == 0) {
#pragma unroll 1
        for (int other = 0; other < TW - 1; ++other) {
          const float* const its = all + (other * 4 + rw) * kOne;
          const floatx2 its_stat = *(const floatx2*)(its + DB * 16 * 64 + 2 * lane);
          const float its_ref = its_stat.x, top = fmaxf(ref, its_ref);
          // without scores so far the sums are zero (or NaN)
          const float mine = ref == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ref - top);
          const float theirs = its_ref == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(its_ref - top);
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
              const floatx4 x = *(const floatx4*)(its + ((d * 4 + r / 4) * 64 + lane) * 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][r + e] = o[d][r + e] * mine + x[e] * theirs;
            }
          sum = sum * mine + its_stat.y * theirs;
          ref = top;
        }
      }
    }
  }

  // The sums to the workspace; parts: of the stream, every step-th work-group from this one on has one.
  __device__ void write(const WidePart& w, int id, int parts, int step, const Layout& l) {
    if (tw) return;
    const Params& a = p.a;
    const int row = rw * 32 + (lane & 31), at = w.row0 + row;
    if (row >= w.rows) return;
    const int member = w.leader + at / a.group;
    const int64_t out = (int64_t)member * a.q_heads + w.head * a.group + at % a.group;
    float* const part = w.c == 0 ? p.prefix_first + out * part_row(DT)
                                 : p.wide_rest + ((int64_t)id * kRows + row) * part_row(DT);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(floatx4*)(part + 32 * d + 2 * r + 4 * hi) = floatx4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
    if (hi == 0) {
      *(floatx2*)(part + DT) = floatx2{ref, sum};
      if (w.c == 0 && l.from[member]) p.prefix_ends[out] = int4{id, parts, row, step};
    }
  }
};

// 64 sequences over 16,384 tokens of 8 key heads of 128 bf16 values, under 256
// rows: 57 us, of which the first 11 go by before a wide stream's first product;
// the matrix cores are busy 26% of it. 16 over 131,000 in e4m3, under 128 rows of
// 8 heads: 139 to 156 us, 39%. (With weights of one term, and an error of 0.0019 in
// place of 0.0017 of the bf16 output's norm: 49 and 112.) 41 in seven groups of 900
// to 12,345, heads of 64: 26.7 us, 4.2 TB/s, waiting for reads 52% of its waves'
// cycles.
template <typename T, bool F8, int DT, bool FULL>
__global__ __launch_bounds__(64 * waves_of(DT), waves_of(DT) / 4) void shared_kernel(Shared p) {
  typedef Wide<T, F8, DT, FULL> W;
  constexpr int NW = W::NW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ Layout l;
  __shared__ uint8_t ok[W::kBuffers][W::TT];
  __shared__ int32_t held[kPages], masked;
  const Params& a = p.a;
  const int team = lay_out<NW, DT>(p, l);
  const int wides = __builtin_amdgcn_readfirstlane(l.totals[0]), thins = __builtin_amdgcn_readfirstlane(l.totals[1]);
  const int total = wides + thins + __builtin_amdgcn_readfirstlane(l.totals[2]);
  // Work-group i runs on XCD i % 8: teams go round the XCDs, a team's members
  // follow each other on one.
  const int rings = gridDim.x % 8 ? 1 : 8, place = blockIdx.x / rings, teams = gridDim.x / rings / team * rings;
  const int me_team = place / team * rings + blockIdx.x % rings, member = place % team, id = me_team * team + member;
  Share share;
  // A wave has at least two tiles, more of long streams: a stream of n tiles takes
  // as long as the tiles of one wave and the join of as many parts as there are
  // waves, least where a wave has about sqrt(n) / 4 (2 sequences over 32,768 tokens
  // of 2 key heads: 48 us with a tile each, 22 with eight). A team has at least a
  // wide tile's units, so that within a stream each has a part, and eight, as it is
  // the whole work-group that begins it.
  int longest = l.longest[0];
#pragma unroll
  for (int k = 1; k < NW; ++k) longest = max(longest, l.longest[k]);
  const int least = max(kLeast, (int)(0.25f * __builtin_amdgcn_sqrtf((float)__builtin_amdgcn_readfirstlane(longest))));
  share.waves = min(max(1, total / (team * max(least, wides ? max(NW, wide_tile(DT)) : 1))), teams);
  share.each = total / share.waves;
  share.more = total % share.waves;
  if (me_team >= share.waves) return;
  const int u0 = share.begin(me_team), u1 = share.begin(me_team + 1);

  const int tile_cost = wide_tile(DT) * team, start_cost = kWideStart * team;
  for (int u = u0; u < min(u1, wides);) {
    const int i = __builtin_amdgcn_readfirstlane(find(l.wide, p.count, u));
    WidePart w;
    w.leader = __builtin_amdgcn_readfirstlane(l.leader[i]);
    w.source = __builtin_amdgcn_readfirstlane(source_of(p, l, i));
    w.tokens = __builtin_amdgcn_readfirstlane(l.from[w.leader]);
    const int m = (__builtin_amdgcn_readfirstlane(l.last[i]) - w.leader + 1) * a.group, blocks = blocks_of(m, team);
    const int tiles = ceil_div(w.tokens, W::TT), cost = start_cost + tiles * tile_cost;
    const int in = u - __builtin_amdgcn_readfirstlane(l.wide[i]), x = in / cost, pos = in - x * cost, begin = u - pos;
    w.head = x / blocks;
    w.row0 = (x % blocks * team + member) * kRows;
    w.rows = min(kRows, m - w.row0);
    const int end = min(cost, pos + (u1 - u));
    w.c = ceil_div(max(0, pos - start_cost), tile_cost);
    w.c1 = ceil_div(max(0, end - start_cost), tile_cost);
    if (w.c < w.c1 && w.rows > 0) {
      W wide{p, lds, ok, held, &masked};
      wide.run(w);
      wide.write(w, id, share.owner(begin + start_cost + (tiles - 1) * tile_cost) - me_team + 1, team, l);
    }
    u += cost - pos;
  }
  __syncthreads();

  // the waves' shares of the rest
  constexpr int VD = DT / 16;
  const int lane = threadIdx.x & 63, g = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // waves of a team that take part: as many in each, so that a stream's are numbered one after the other
  const int waves = min(max(1, share.each / least), team * NW);
  const int x0 = max(u0, wides), span = u1 - x0;
  if (span <= 0) return;
  // n units go to the last min(n, waves) waves of a team: only where the wide
  // streams end there are fewer, and the next one's first wave goes on with what
  // the last of them began
  const auto wave_begin = [&](int64_t n, int k) { return (int)(n * k / min(n, (int64_t)waves)); };
  const auto owner = [&](int u) {  // the wave that has unit u
    const int of = share.owner(u), begin = max(share.begin(of), wides), n = share.begin(of + 1) - begin;
    int k = (int)((int64_t)(u - begin) * min(n, waves) / n);
    while (wave_begin(n, k + 1) <= u - begin) ++k;
    return of * waves + waves - min(n, waves) + k;
  };
  const int at_wave = wave * team + member, mine = at_wave - (waves - min(span, waves));
  if (mine < 0 || at_wave >= waves) return;
  const int me = me_team * waves + at_wave, a1 = x0 + wave_begin(span, mine + 1);
  for (int u = x0 + wave_begin(span, mine); u < a1;) {
    Span sp{};
    Stream at;
    const char* q_row;
    int pos, first_seq;
    const bool thin = u < wides + thins;
    if (thin) {
      const int i = __builtin_amdgcn_readfirstlane(find(l.thin, p.count, u - wides));
      const int leader = __builtin_amdgcn_readfirstlane(l.leader[i]);
      sp.end = __builtin_amdgcn_readfirstlane(l.from[leader]);
      sp.tiles = ceil_div(sp.end, kTile), sp.cost = kStart + sp.tiles;
      const int in = u - wides - __builtin_amdgcn_readfirstlane(l.thin[i]), head = in / sp.cost;
      pos = in - head * sp.cost;
      first_seq = leader;
      at = Stream{__builtin_amdgcn_readfirstlane(source_of(p, l, i)), head, (__builtin_amdgcn_readfirstlane(l.last[i]) - leader + 1) * a.group, head * a.group, head};
      q_row = a.q + ((p.first + leader + i16 / a.group) * a.q_stride + (at.q_head + i16 % a.group) * a.q_head) * 2;
    } else {
      const int i = __builtin_amdgcn_readfirstlane(find(l.own, p.count, u - wides - thins));
      sp.begin = __builtin_amdgcn_readfirstlane(l.from[i]), sp.base = sp.begin & ~7, sp.end = __builtin_amdgcn_readfirstlane(l.len[i]);
      sp.tiles = max(1, ceil_div(sp.end - sp.base, kTile)), sp.cost = kStart + sp.tiles;
      const int in = u - wides - thins - __builtin_amdgcn_readfirstlane(l.own[i]), x = in / sp.cost;
      pos = in - x * sp.cost;
      first_seq = i;
      at = stream_of(a, p.first + i, x / a.head_tiles, x % a.head_tiles);
      q_row = query_of(a, at, i16);
    }
    const int c = max(0, pos - kStart), c1 = max(0, min(sp.cost, pos + (a1 - u)) - kStart);
    if (c < c1) {
      const Sums<DT> s = attend_tiles<T, F8, DT, false, FULL, kStage>(p.a, sp, at, q_row, c, c1, (int64_t*)lds + wave * kStage);
      if (i16 < at.heads) {
        const int seq = first_seq + (thin ? i16 / a.group : 0);
        const int64_t out = (int64_t)seq * a.q_heads + at.q_head + (thin ? i16 % a.group : i16);
        float* const part = c ? p.wave_rest + ((int64_t)me * kHeads + i16) * part_row(DT)
                              : (thin ? p.prefix_first : p.own_first) + out * part_row(DT);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < VD; j += 4)
            *(floatx4*)(part + dim_of<F8, DT>(g, j, r)) = floatx4{s.o[j][r], s.o[j + 1][r], s.o[j + 2][r], s.o[j + 3][r]};
        if (g == 0) {
          *(floatx2*)(part + DT) = floatx2{s.ref, s.sum};
          if (c == 0) {
            const int parts = owner(u - pos + sp.cost - 1) - me + 1;
            if (!thin) p.own_ends[out] = int2{me, parts};
            if (thin && l.from[seq]) p.prefix_ends[out] = int4{me, parts, i16, 0};
            if (!thin && sp.begin == 0) p.prefix_ends[out] = int4{0, 0, 0, 0};
          }
        }
      }
    }
    u += sp.cost - pos;
  }
}

// Joins the parts of a query row: a thread has four dims of every kAtOnce-th part.
// Bound by its chain of three reads (ends, parts, output): 4.0 to 7.6 us.
template <typename T, int DT>
__global__ __launch_bounds__(kJoin) void join_kernel(Shared p) {
  constexpr int kLanes = DT / 4, kAtOnce = kJoin / kLanes, kLoads = 8;
  __shared__ float weight[kGroups * (1 + 2 * waves_of(DT))];
  __shared__ float tops[kJoin / 64], tots[kJoin / 64];
  __shared__ floatx4 sums[kAtOnce][kLanes];
  const Params& a = p.a;
  const int64_t out = blockIdx.x;
  const int4 prefix = p.prefix_ends[out];
  const int2 own = p.own_ends[out];
  const int n_prefix = prefix.y, parts = n_prefix + own.y;
  const int head = (int)(out % a.q_heads);
  const auto part = [&](int i) -> const float* {
    if (i < n_prefix) {
      if (i == 0) return p.prefix_first + out * part_row(DT);
      return prefix.w ? p.wide_rest + ((int64_t)(prefix.x + i * prefix.w) * kRows + prefix.z) * part_row(DT)
                      : p.wave_rest + ((int64_t)(prefix.x + i) * kHeads + prefix.z) * part_row(DT);
    }
    i -= n_prefix;
    if (i == 0) return p.own_first + out * part_row(DT);
    return p.wave_rest + ((int64_t)(own.x + i) * kHeads + head % a.group % kHeads) * part_row(DT);
  };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lane4 = threadIdx.x % kLanes, row = threadIdx.x / kLanes, d = 4 * lane4;
  floatx4 y[kLoads];
  const auto fetch = [&](int i0) {
#pragma unroll
    for (int e = 0; e < kLoads; ++e)
      if (i0 + e * kAtOnce < parts) y[e] = *(const floatx4*)(part(i0 + e * kAtOnce) + d);
  };
  fetch(row);  // on their way while the weights are found
  float top = -__builtin_inff();
  for (int i = threadIdx.x; i < parts; i += kJoin) {
    const float m = part(i)[DT];
    weight[i] = m;
    top = fmaxf(top, m);
  }
  for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  float tot = 0;
  for (int i = threadIdx.x; i < parts; i += kJoin) {
    const float m = weight[i];
    const float f = m == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - top);  // then its sums are zero (or NaN)
    weight[i] = f;
    tot += f * part(i)[DT + 1];
  }
  for (int m = 32; m; m >>= 1) tot += __shfl_xor(tot, m, 64);
  if (lane == 0) tots[wave] = tot;
  __syncthreads();
  tot = (tots[0] + tots[1]) + (tots[2] + tots[3]);
  floatx4 acc = {0, 0, 0, 0};
  for (int i0 = row; i0 < parts; i0 += kAtOnce * kLoads) {
    if (i0 != row) fetch(i0);
#pragma unroll
    for (int e = 0; e < kLoads; ++e) {
      const int i = i0 + e * kAtOnce;
      if (i < parts) acc += y[e] * weight[i];
    }
  }
  sums[row][lane4] = acc;
  __syncthreads();
  if (row) return;
  for (int r = 1; r < kAtOnce; ++r) acc += sums[r][lane4];
  const int64_t at = (int64_t)p.first * a.q_heads + out;
  const float inv = (a.v_scale ? a.v_scale[head / a.group] : 1.f) / tot;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = tot == 0.f ? 0.f : acc[e] * inv;
  if (d < a.dim) *(uintx2*)(a.out + (at * a.dim + d) * 2) = uintx2{pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3])};
  if (d == 0 && a.lse) a.lse[at] = tot == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(tot)) * kLn2;
}

// How a call's work is laid out, from its sizes alone.
struct Plan {
  int dt, group, head_tiles;
  int64_t work_groups;
  int64_t ends, firsts, wide_rest, wave_rest, bytes;  // of the workspace: bytes of each
};

Plan plan_of(int64_t batch, int64_t q_heads, const KvPages& pages, int64_t max_len) {
  Plan a;
  a.dt = pages.dim <= 64 ? 64 : pages.dim <= 128 ? 128 : 256;
  a.group = (int)(q_heads / pages.heads);
  a.head_tiles = (a.group + kHeads - 1) / kHeads;
  const int64_t count = std::min<int64_t>(batch, kBatch);
  // Units of a launch, at most: what a prefix of n tiles under more than 16 rows
  // costs, a quarter more with teams, is no more than its members would cost for
  // themselves, n for each 16 of their rows, but for its start and its last tile.
  const int64_t tiles = max_len / kTile + 2 + kStart;
  const int64_t start = (kTeam + a.group / kRows + 2) * (kWideStart + wide_tile(a.dt));
  const int64_t most = 0x7FFFFFFF / std::max<int64_t>(1, count * pages.heads);  // of a sequence's streams to a key head
  if (tiles > most || tiles * a.head_tiles > most - start) throw std::invalid_argument("batch x heads x tokens is too large");
  if (count * q_heads * kJoin > 0xFFFFFFFFll) throw std::invalid_argument("batch x heads is too large");  // threads of the joining launch
  a.work_groups = kGroups;  // those without units end at once
  const int64_t rows = count * q_heads, row = part_row(a.dt) * 4;
  a.ends = rows * 24, a.firsts = rows * row;
  a.wide_rest = a.work_groups * kRows * row;
  a.wave_rest = a.work_groups * waves_of(a.dt) * kHeads * row;
  a.bytes = (a.ends + 15) / 16 * 16 + 2 * a.firsts + a.wide_rest + a.wave_rest;
  return a;
}

template <typename T, bool F8, int DT>
void launch(const Shared& p, const Plan& plan, hipStream_t s) {
  auto kernel = p.a.dim == DT ? shared_kernel<T, F8, DT, true> : shared_kernel<T, F8, DT, false>;
  constexpr int lds = std::max(Wide<T, F8, DT, true>::kLds, waves_of(DT) * kStage * 8);
  hip_check(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "shared attention");
  kernel<<<(unsigned)plan.work_groups, 64 * waves_of(DT), lds, s>>>(p);
  hip_check(hipGetLastError(), "shared attention");
  join_kernel<T, DT><<<(unsigned)(p.count * p.a.q_heads), kJoin, 0, s>>>(p);
  hip_check(hipGetLastError(), "shared attention join");
}

template <typename T, bool F8>
void launch_dim(const Shared& p, const Plan& plan, hipStream_t s) {
  if (plan.dt == 64) launch<T, F8, 64>(p, plan, s);
  else if (plan.dt == 128) launch<T, F8, 128>(p, plan, s);
  else launch<T, F8, 256>(p, plan, s);
}

}  // namespace

int64_t shared_workspace(int64_t batch, int64_t q_heads, const KvPages& pages, int64_t max_len) {
  return batch ? plan_of(batch, q_heads, pages, max_len).bytes : 0;
}

void shared_attend(const AttendArgs& a, const int32_t* groups, const int32_t* shared, int64_t n_groups, const KvPages& pages,
                   hipStream_t s) {
  if (a.batch == 0) return;
  const int64_t width = (int64_t)a.table_width << pages.page_shift;
  Shared p{};
  Params& r = p.a;
  r.limit = pages.pages ? (int)std::min<int64_t>({a.max_len, width, 0x7FFFFF00}) : 0;
  const Plan plan = plan_of(a.batch, a.q.heads, pages, a.max_len);
  if (a.workspace_bytes < plan.bytes || !a.workspace || ((uintptr_t)a.workspace & 15u))
    throw std::invalid_argument("workspace must be 16-byte aligned and hold " + std::to_string(plan.bytes) + " bytes");
  r.q = (const char*)a.q.p, r.q_stride = a.q.stride, r.q_head = a.q.head_stride;
  r.k = pages.k, r.v = pages.v;
  r.page_stride = pages.page_stride, r.head_stride = pages.head_stride, r.row_stride = pages.row_stride;
  r.tables = a.tables, r.table_stride = a.table_stride, r.lens = a.lens;
  r.k_scale = pages.k_scale, r.v_scale = pages.v_scale;
  r.out = (char*)a.out, r.lse = a.lse;
  r.scale = a.scale * 1.4426950408889634f;
  r.batch = (int)a.batch, r.heads = pages.heads, r.q_heads = a.q.heads, r.lists = pages.heads;
  r.group = plan.group, r.head_tiles = plan.head_tiles, r.side = 1;
  r.page_shift = pages.page_shift, r.pages = pages.pages, r.dim = pages.dim;
  p.groups = groups, p.shared = shared, p.n_groups = (int)n_groups;
  p.far = pages.row_stride > 0x3FFFFFFF / pages.page;
  char* w = (char*)a.workspace;
  const int64_t rows = plan.ends / 24;
  p.prefix_ends = (int4*)w, p.own_ends = (int2*)(w + rows * 16);
  w += (plan.ends + 15) / 16 * 16;
  p.prefix_first = (float*)w, p.own_first = (float*)(w + plan.firsts);
  p.wide_rest = (float*)(w + 2 * plan.firsts), p.wave_rest = (float*)(w + 2 * plan.firsts + plan.wide_rest);
  for (p.first = 0; p.first < a.batch; p.first += kBatch) {
    p.count = (int)std::min<int64_t>(kBatch, a.batch - p.first);
    if (pages.type == kE4M3) {
      if (a.type == kF16) launch_dim<f16, true>(p, plan, s);
      else launch_dim<bf16, true>(p, plan, s);
    } else if (a.type == kF16) {
      launch_dim<f16, false>(p, plan, s);
    } else {
      launch_dim<bf16, false>(p, plan, s);
    }
  }
}

}  // namespace jasper_amd
