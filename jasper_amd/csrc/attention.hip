// attention.hip -- attention of one new token per sequence over the paged
// cache: over all its tokens (or the last ones), and over the first, the last
// and a list of ids in between.
#include "kvcache.hpp"

#include "attend.hpp"
#include "graph.hpp"
#include "kvtypes.hpp"

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <type_traits>

namespace jasper_amd {

namespace {

using namespace attention;

constexpr int kWaves = 2048;  // at most; of a call
constexpr int kStage = 512;   // row offsets of a wave, in LDS
constexpr int kJoin = 256;   // threads of a joining work-group
constexpr int kGroupStage = 256;        // row offsets of a wave of a group, in LDS
constexpr int kGroupLds = 64 << 10;     // bytes at most
// waves of a group at most. A compute unit has registers for 16 and more of 64
// values, for four of 256; of 128 for eight of the largest form (169 of a lane)
// and for 12 to 16 of the others, which was not tried
constexpr int group_waves(int dt) { return dt == 64 ? 16 : dt == 128 ? 8 : 4; }
// A wave's sums in the workspace: dt floats and two for each of its heads, and
// what keeps the next one's on 16 bytes.
__host__ __device__ constexpr int part_size(int heads, int dt) { return (heads * (dt + 2) + 3) / 4 * 4; }

// Every wave adds up the lengths for itself (lane i a run of sequences) and
// finds the sequence its first unit lies in, and the units of one stream
// before that sequence. -1: there is no work for it.
template <bool LISTED>
__device__ int find_sequence(const Params& p, int streams, Share& share, int& before) {
  const int lane = threadIdx.x & 63;
  const int run = (p.batch + 63) / 64;
  const int b0 = min(lane * run, p.batch), b1 = min(b0 + run, p.batch);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += span_of<LISTED>(p, b).cost;
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  const int total = __builtin_amdgcn_readlane(incl, 63) * streams;  // known to be the same in all lanes
  share.waves = min(total, (int)gridDim.x);
  share.each = total / share.waves;
  share.more = total % share.waves;
  if ((int)blockIdx.x >= share.waves) return -1;
  const int at = share.begin(blockIdx.x) / streams;  // unit of a stream, were the streams side by side
  const int src = __ffsll((unsigned long long)__ballot(at < incl)) - 1;
  int pre = incl - mine, b = b0;
  if (lane == src) {
    for (;; ++b) {
      const int n = span_of<LISTED>(p, b).cost;
      if (at < pre + n) break;
      pre += n;
    }
  }
  before = __builtin_amdgcn_readlane(pre, src);
  return __builtin_amdgcn_readlane(b, src);
}

// The work is shared out evenly over the waves that a GPU holds at once:
// every work-group is one wave with an equal run of the units of all
// sequences and streams, so that waves in different phases (finding their
// rows, streaming, writing) share a compute unit without waiting for each
// other. A stream that one wave has whole is finished here, the others' parts
// go to the workspace: a wave has at most one that an earlier wave began (slot
// 0) and one that it begins itself (slot 1).
//
// Bound by the rows' reads: 48 sequences of 17 to 8192 bf16 tokens under 32 / 8
// heads 48.7 us (5.6 TB/s), four of 131k e4m3 tokens 174 us (6.2; a kernel that
// only reads 6.2 to 6.4); matrix cores 5 and 11 % busy. A shorter call is its
// chain of reads: lengths, table, rows (700 tokens 5.6 us).
//
// More than 16 query heads to a list are further waves of the work-group,
// which take the same rows at about the same time and find them in the caches:
// 64 sequences of 8192 tokens, one key head of 128 values under 64 heads, 104
// us (183 with a work-group for each 16; under 32 heads 75 and 101).
constexpr int side_of(int dt) { return dt == 256 ? 4 : 8; }

template <typename T, bool F8, int DT, bool LISTED, bool FULL>
__global__ __launch_bounds__(64 * (FULL ? 1 : side_of(DT)), DT == 256 ? 1 : 2) void attend_kernel(Params p) {
  constexpr int VD = DT / 16;
  extern __shared__ __attribute__((aligned(16))) int64_t lds[];
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int wave = FULL ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_list = (p.head_tiles + p.side - 1) / p.side, streams = p.lists * per_list;
  Share share;
  int before;
  int b = find_sequence<LISTED>(p, streams, share, before);
  if (b < 0) return;
  int u = share.begin(blockIdx.x);
  const int u1 = share.begin(blockIdx.x + 1);
  Span sp = span_of<LISTED>(p, b);
  int x = (u - before * streams) / sp.cost;
  int pos = (u - before * streams) % sp.cost;

  for (; u < u1; u += sp.cost - pos, pos = 0, ++x) {
    if (x == streams) {
      x = 0;
      sp = span_of<LISTED>(p, ++b);
    }
    const int list = x / per_list, head_tile = x % per_list * p.side + wave;
    const int c = max(0, pos - kStart), c1 = max(0, min(sp.cost, pos + (u1 - u)) - kStart);
    if (c1 == c || head_tile >= p.head_tiles) continue;
    const Stream at = stream_of(p, b, list, head_tile);
    const Sums<DT> s = attend_tiles<T, F8, DT, LISTED, FULL, kStage>(p, sp, at, query_of(p, at, i), c, c1, lds + wave * kStage);
    if (c == 0 && lane == 0)
      p.ends[((int64_t)b * p.lists + list) * p.head_tiles + head_tile] =
          int2{(int)blockIdx.x, share.owner(u - pos + sp.cost - 1)};
    if (i >= at.heads) continue;
    if (c == 0 && c1 == sp.tiles) {
      const int64_t row = (int64_t)b * p.q_heads + at.q_head + i;
      const float inv = (p.v_scale ? p.v_scale[at.kv_head] : 1.f) / s.sum;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int j = 0; j < VD; j += 4) {
          const int d = dim_of<F8, DT>(g, j, r);
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = s.sum == 0.f ? 0.f : s.o[j + e][r] * inv;
          if (FULL || d < p.dim) *(uintx2*)(p.out + (row * p.dim + d) * 2) = uintx2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
        }
      }
      if (g == 0 && p.lse) p.lse[row] = s.sum == 0.f ? -__builtin_inff() : (s.ref + __builtin_amdgcn_logf(s.sum)) * kLn2;
    } else {
      float* part = p.parts + (((int64_t)blockIdx.x * 2 + (c == 0 ? 1 : 0)) * p.side + wave) * part_size(p.part_heads, DT);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VD; j += 4)
          *(floatx4*)(part + i * DT + dim_of<F8, DT>(g, j, r)) = floatx4{s.o[j][r], s.o[j + 1][r], s.o[j + 2][r], s.o[j + 3][r]};
      if (g == 0) *(floatx2*)(part + p.part_heads * DT + 2 * i) = floatx2{s.ref, s.sum};
    }
  }
}

// Short streams: a work-group has a stream, its waves equal runs of the tiles,
// and joins them itself. No lengths to add up and no second kernel.
template <typename T, bool F8, int DT, bool LISTED, bool FULL>
__global__ __launch_bounds__(64 * group_waves(DT)) void attend_group_kernel(Params p) {
  constexpr int VD = DT / 16;
  extern __shared__ __attribute__((aligned(16))) int64_t lds[];
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int head_tile = blockIdx.x % p.head_tiles, list = blockIdx.x / p.head_tiles % p.lists;
  const int b = blockIdx.x / p.head_tiles / p.lists;
  const Span sp = span_of<LISTED>(p, b);
  const Stream at = stream_of(p, b, list, head_tile);
  const Sums<DT> s = attend_tiles<T, F8, DT, LISTED, FULL, kGroupStage>(
      p, sp, at, query_of(p, at, i), sp.tiles * wave / waves, sp.tiles * (wave + 1) / waves, lds + wave * kGroupStage);
  __syncthreads();  // the rows' offsets make room for the waves' sums
  float* const sums = (float*)lds;                        // [waves][heads][DT]
  floatx2* const stats = (floatx2*)(sums + waves * at.heads * DT);  // [waves][heads]
  if (i < at.heads) {
    float* mine = sums + (wave * at.heads + i) * DT;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < VD; j += 4)
        *(floatx4*)(mine + dim_of<F8, DT>(g, j, r)) = floatx4{s.o[j][r], s.o[j + 1][r], s.o[j + 2][r], s.o[j + 3][r]};
    if (g == 0) stats[wave * at.heads + i] = floatx2{s.ref, s.sum};
  }
  __syncthreads();
  for (int e = threadIdx.x; e < at.heads * (DT / 4); e += blockDim.x) {
    const int n = e / (DT / 4), d = e % (DT / 4) * 4;
    float top = stats[n].x, tot = 0;
    for (int w = 1; w < waves; ++w) top = fmaxf(top, stats[w * at.heads + n].x);
    floatx4 acc = {0, 0, 0, 0};
    for (int w = 0; w < waves; ++w) {
      const floatx2 m = stats[w * at.heads + n];
      const float f = m.x == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m.x - top);  // then its sums are zero (or NaN)
      tot += f * m.y;
      acc += *(const floatx4*)(sums + (w * at.heads + n) * DT + d) * f;
    }
    const int64_t row = (int64_t)b * p.q_heads + at.q_head + n;
    const float inv = (p.v_scale ? p.v_scale[at.kv_head] : 1.f) / tot;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = tot == 0.f ? 0.f : acc[k] * inv;
    if (FULL || d < p.dim) *(uintx2*)(p.out + (row * p.dim + d) * 2) = uintx2{pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3])};
    if (d == 0 && p.lse) p.lse[row] = tot == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(tot)) * kLn2;
  }
}

// Joins the parts of a stream that several waves had: a work-group per
// sequence, stream, head and DIMS dims. The parts' weights go to LDS, then a thread has four dims of every
// kRows-th part, eight loads in flight. A launch and two reads in a row: 4.4 us
// for 8 streams of 22 parts, 4.9 for 384 of up to 10.
template <typename T, int DT, int DIMS>
__global__ __launch_bounds__(kJoin) void join_kernel(Params p) {
  const int head_tile = blockIdx.x % p.head_tiles, list = blockIdx.x / p.head_tiles % p.lists, n = blockIdx.y;
  const int b = blockIdx.x / p.head_tiles / p.lists, head0 = head_tile * kHeads;
  if (n >= p.group - head0) return;
  const int2 range = p.ends[blockIdx.x];
  const int parts = range.y - range.x + 1;
  if (parts == 1) return;
  constexpr int kLanes = DIMS / 4, kRows = kJoin / kLanes, kBatch = 8;
  __shared__ float weight[kWaves];
  __shared__ float tops[kJoin / 64], tots[kJoin / 64];
  __shared__ floatx4 sums[kRows][kLanes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int size = part_size(p.part_heads, DT), stats = p.part_heads * DT + 2 * n;
  // the part that begins the stream, and what part i > 0 is i steps from
  const float* const own = p.parts + (((int64_t)range.x * 2 + 1) * p.side + head_tile % p.side) * size;
  const float* const rest = own - p.side * size;
  const auto part = [&](int i) { return i ? rest + (int64_t)i * 2 * p.side * size : own; };
  const int lane4 = threadIdx.x % kLanes, row = threadIdx.x / kLanes, d = blockIdx.z * DIMS + 4 * lane4;
  floatx4 y[kBatch];
  const auto fetch = [&](int i0) {
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const int i = i0 + e * kRows;
      if (i < parts) y[e] = *(const floatx4*)(part(i) + n * DT + d);
    }
  };
  fetch(row);  // on their way while the weights are found
  float top = -__builtin_inff();
  for (int i = threadIdx.x; i < parts; i += kJoin) {
    const float m = part(i)[stats];
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
    tot += f * part(i)[stats + 1];
  }
  for (int m = 32; m; m >>= 1) tot += __shfl_xor(tot, m, 64);
  if (lane == 0) tots[wave] = tot;
  __syncthreads();
  tot = (tots[0] + tots[1]) + (tots[2] + tots[3]);
  floatx4 acc = {0, 0, 0, 0};
  for (int i0 = row; i0 < parts; i0 += kRows * kBatch) {
    if (i0 != row) fetch(i0);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const int i = i0 + e * kRows;
      if (i < parts) acc += y[e] * weight[i];
    }
  }
  sums[row][lane4] = acc;
  __syncthreads();
  if (row) return;
  for (int r = 1; r < kRows; ++r) acc += sums[r][lane4];
  const int64_t at = (int64_t)b * p.q_heads + list * p.group + head0 + n;
  const float inv = (p.v_scale ? p.v_scale[list * p.heads / p.lists] : 1.f) / tot;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = tot == 0.f ? 0.f : acc[e] * inv;
  if (d < p.dim) *(uintx2*)(p.out + (at * p.dim + d) * 2) = uintx2{pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3])};
  if (d == 0 && p.lse) p.lse[at] = tot == 0.f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(tot)) * kLn2;
}

int compute_units() {
  static const int n = [] {
    int device = 0, v = 0;
    hip_check(hipGetDevice(&device), "get device");
    hip_check(hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, device), "device attribute");
    return v > 0 ? v : 256;
  }();
  return n;
}

// How a call's work is laid out, from its sizes alone.
struct Plan {
  int dt, lists, group, head_tiles, side, part_heads;
  int64_t streams, work_groups;
  int group_waves;  // of a group's work-group; 0: the waves share all streams
  bool joins;
  int64_t ends_bytes, bytes;
};

Plan plan_of(int64_t batch, int64_t q_heads, const KvPages& pages, int64_t max_tokens, int64_t lists) {
  Plan a;
  a.dt = pages.dim <= 64 ? 64 : pages.dim <= 128 ? 128 : 256;
  a.lists = (int)(lists ? lists : pages.heads);
  a.group = (int)(q_heads / a.lists);
  a.head_tiles = (a.group + kHeads - 1) / kHeads;
  a.side = std::min(a.head_tiles, side_of(a.dt));
  a.part_heads = std::min(a.group, kHeads);
  a.streams = (int64_t)a.lists * a.head_tiles;
  // a window's first group of 8 rows may start 7 tokens early
  const int64_t tiles = std::max<int64_t>(1, max_tokens / kTile + (max_tokens % kTile + (lists ? 0 : 7) + kTile - 1) / kTile);
  if (tiles + kStart > 0x7FFFFFFF / std::max<int64_t>(1, batch * a.streams)) throw std::invalid_argument("batch x heads x tokens is too large");
  const int64_t resident = std::min(kWaves, compute_units() * (a.dt == 256 ? 4 : 8));
  // A group spares the second kernel, but its compute unit reads a tile of each
  // wave in 1.4 us (90 GB/s) while most of the GPU idles where there are few
  // streams. Of 8 key
  // heads of 128 fp16 values, group against shared, us: one sequence of 100
  // tokens 5.2 / 8.4, 300 7.9 / 8.5, 700 10.8 / 8.9; four of 500 9.2 / 10.1, of
  // 1000 17.1 / 12.5; 16 of 1000 20.4 / 21.5; 64 of 1000 45.7 / 54.4; 512 of 128
  // 48.7 / 57.2. Longer tables may hold sequences too unlike for it; lists are
  // alike, and are grouped up to eight tiles a wave where there is one for
  // three in four compute units: 1,068 tokens in 128 lists 29.3 / 26.3, in 256
  // 30.2 / 37.7, in 512 54.1 / 64.2; 1,272 tokens in 192 lists 28.6 / 33. Between
  // 128 and 192 neither was measured: the cut may lie lower (near 165, if the
  // times change evenly). The waves are counted as the shared kernel's, eight to
  // a compute unit; groups of 64 values have room for twice as many, not tried:
  // 204 streams of up to 1000 tokens get ten waves each, with up to four tiles
  // in a row, 11.8 us.
  const int64_t all = batch * a.streams;
  const int most = std::min(group_waves(a.dt), kGroupLds / std::max(a.part_heads * (a.dt + 2) * 4, kGroupStage * 8));
  const int each = lists && 4 * all >= 3 * compute_units() ? 8 : 2 * all >= compute_units() ? 4 : 2;
  const bool grouped = all > 0 && tiles <= most * each;
  a.group_waves = grouped ? (int)std::clamp<int64_t>(resident / all, 1, std::min<int64_t>(most, tiles)) : 0;
  if (a.group_waves) {
    a.joins = false, a.work_groups = 0, a.ends_bytes = 0, a.bytes = 0;
    return a;
  }
  // Fewer waves where there is little for each, by what was measured of small
  // calls in us: a tile more costs a wave 1.2, a part more the join of its
  // stream 0.02, a wave more the call 0.003. One sequence of 16,000 tokens 24.9
  // -> 19.6 (2048 waves before), 131,072 under one key head 58.9 -> 22.8.
  const int64_t shared = batch * a.lists * ((a.head_tiles + a.side - 1) / a.side);
  const double units = (double)shared * (tiles + kStart);
  const double cost = (0.02 / shared + 0.003 * a.side) * std::max(1.0, a.part_heads / 8.0);
  const int64_t worth = std::max<int64_t>(1, (int64_t)std::sqrt(1.2 * units / cost));
  a.work_groups = std::min({(int64_t)units, resident / a.side, worth});
  a.joins = tiles > 1;
  a.ends_bytes = (batch * a.streams * 8 + 15) / 16 * 16;
  a.bytes = a.ends_bytes + a.work_groups * 2 * a.side * part_size(a.part_heads, a.dt) * 4;
  return a;
}

template <typename T, bool F8, int DT>
void launch(const Params& p, const Plan& plan, bool listed, hipStream_t s) {
  const bool full = p.dim == DT;
  if (plan.group_waves) {
    auto kernel = listed ? (full ? attend_group_kernel<T, F8, DT, true, true> : attend_group_kernel<T, F8, DT, true, false>)
                         : (full ? attend_group_kernel<T, F8, DT, false, true> : attend_group_kernel<T, F8, DT, false, false>);
    const size_t lds = (size_t)plan.group_waves * std::max(plan.part_heads * (DT + 2) * 4, kGroupStage * 8);
    kernel<<<(unsigned)(p.batch * plan.streams), 64 * plan.group_waves, lds, s>>>(p);
    hip_check(hipGetLastError(), "attention");
    return;
  }
  const bool alone = full && plan.side == 1;
  auto kernel = listed ? (alone ? attend_kernel<T, F8, DT, true, true> : attend_kernel<T, F8, DT, true, false>)
                       : (alone ? attend_kernel<T, F8, DT, false, true> : attend_kernel<T, F8, DT, false, false>);
  kernel<<<(unsigned)plan.work_groups, 64 * plan.side, plan.side * kStage * 8, s>>>(p);
  hip_check(hipGetLastError(), "attention");
  if (plan.joins) {
    const int64_t all = p.batch * plan.streams;
    // Few streams: more work-groups with 32 dims each (131,072 tokens under one
    // key head 22.8 us, 27.7 without; of 32 streams under 8 heads, where there
    // are work-groups enough, 189 and 176).
    if (4 * all * plan.part_heads <= compute_units())
      join_kernel<T, DT, 32><<<dim3((unsigned)all, (unsigned)plan.part_heads, DT / 32), kJoin, 0, s>>>(p);
    else
      join_kernel<T, DT, DT><<<dim3((unsigned)all, (unsigned)plan.part_heads), kJoin, 0, s>>>(p);
    hip_check(hipGetLastError(), "attention join");
  }
}

template <typename T, bool F8>
void launch_dim(const Params& p, const Plan& plan, bool listed, hipStream_t s) {
  if (plan.dt == 64) launch<T, F8, 64>(p, plan, listed, s);
  else if (plan.dt == 128) launch<T, F8, 128>(p, plan, listed, s);
  else launch<T, F8, 256>(p, plan, listed, s);
}

}  // namespace

int64_t attend_workspace(int64_t batch, int64_t q_heads, const KvPages& pages, int64_t max_tokens, int64_t lists) {
  return batch ? plan_of(batch, q_heads, pages, max_tokens, lists).bytes : 0;
}

void attend(const AttendArgs& a, const KvPages& pages, hipStream_t s) {
  if (a.batch == 0) return;
  const int64_t width = (int64_t)a.table_width << pages.page_shift;
  const bool listed = a.lists != 0;
  Params p{};
  p.limit = pages.pages ? (int)std::min<int64_t>({a.max_len, width, 0x7FFFFF00}) : 0;
  const int64_t most = listed ? a.first + a.last + a.count : a.last < 0 ? a.max_len : std::min(a.max_len, a.last);
  const Plan plan = plan_of(a.batch, a.q.heads, pages, most, a.lists);
  if (plan.bytes && (a.workspace_bytes < plan.bytes || !a.workspace || ((uintptr_t)a.workspace & 15u)))
    throw std::invalid_argument("workspace must be 16-byte aligned and hold " + std::to_string(plan.bytes) + " bytes");
  p.q = (const char*)a.q.p, p.q_stride = a.q.stride, p.q_head = a.q.head_stride;
  p.k = pages.k, p.v = pages.v;
  p.page_stride = pages.page_stride, p.head_stride = pages.head_stride, p.row_stride = pages.row_stride;
  p.tables = a.tables, p.table_stride = a.table_stride, p.lens = a.lens, p.ids = a.ids;
  p.k_scale = pages.k_scale, p.v_scale = pages.v_scale;
  p.out = (char*)a.out, p.lse = a.lse;
  p.ends = (int2*)a.workspace, p.parts = (float*)((char*)a.workspace + plan.ends_bytes);
  p.scale = a.scale * 1.4426950408889634f;
  p.batch = (int)a.batch, p.heads = pages.heads, p.q_heads = a.q.heads;
  p.lists = plan.lists, p.group = plan.group, p.head_tiles = plan.head_tiles, p.side = plan.side, p.count = pages.pages ? a.count : 0;
  p.page_shift = pages.page_shift, p.pages = pages.pages, p.dim = pages.dim;
  p.first = (int)a.first, p.last = (int)std::min<int64_t>(a.last, 0x7FFFFF00), p.part_heads = plan.part_heads;
  if (pages.type == kE4M3) {
    if (a.type == kF16) launch_dim<f16, true>(p, plan, listed, s);
    else launch_dim<bf16, true>(p, plan, listed, s);
  } else if (a.type == kF16) {
    launch_dim<f16, false>(p, plan, listed, s);
  } else {
    launch_dim<bf16, false>(p, plan, listed, s);
  }
}

}  // namespace jasper_amd
