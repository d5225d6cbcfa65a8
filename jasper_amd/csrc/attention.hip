// attention.hip -- attention of one new token per sequence over the paged
// cache: over all its tokens (or the last ones), and over the first, the last
// and a list of ids in between.
#include "kvcache.hpp"

#include "graph.hpp"
#include "kvtypes.hpp"

#include <algorithm>
#include <stdexcept>

namespace jasper_amd {

namespace {

constexpr int kMaxDim = 256;

// A work-group of four waves per sequence and query head; a wave takes every
// fourth token, a lane four of the dims, with the softmax's running maximum
// and sum per wave, joined at the end.
template <typename T, typename CT>
__global__ __launch_bounds__(256) void attend_kernel(AttendArgs a, KvPages pages) {
  const int64_t b = blockIdx.x;
  const int hq = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = a.q.heads / pages.heads, h = hq / group;
  const int64_t width = (int64_t)a.table_width << pages.page_shift;
  const int64_t limit = a.max_len < width ? a.max_len : width;
  int64_t len = a.lens[b];
  len = len < 0 ? 0 : len > limit ? limit : len;
  const int64_t first = a.lists ? (a.first < len ? a.first : len) : 0;
  int64_t last = a.last < 0 ? 0 : len - a.last;
  if (last < first) last = first;
  const int64_t always = first + (len - last);
  const int64_t total = always + a.count;
  const int32_t* ids = a.lists ? a.ids + ((int64_t)b * a.lists + hq / (a.q.heads / a.lists)) * a.count : nullptr;
  const bool mine = lane * 4 < pages.dim;
  float q[4] = {0, 0, 0, 0}, acc[4] = {0, 0, 0, 0};
  if (mine) widen(*(const Pack<T, 4>*)((const T*)a.q.p + b * a.q.stride + hq * a.q.head_stride + lane * 4), q);
  const float ks = pages.k_scale ? pages.k_scale[h] : 1.f, vs = pages.v_scale ? pages.v_scale[h] : 1.f;
  float top = -__builtin_inff(), sum = 0;
  for (int64_t i = wave; i < total; i += 4) {
    int64_t t = i < first ? i : i < always ? last + (i - first) : ids[i - always];
    if (i >= always && (t < first || t >= last)) continue;
    const int32_t page = a.tables[b * a.table_stride + (t >> pages.page_shift)];
    if (page < 0 || page >= pages.pages) continue;
    const int64_t off = page * pages.page_stride + h * pages.head_stride +
                        (t & (pages.page - 1)) * pages.row_stride + lane * 4;
    float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
    if (mine) {
      widen(*(const Pack<CT, 4>*)((const CT*)pages.k + off), k);
      widen(*(const Pack<CT, 4>*)((const CT*)pages.v + off), v);
    }
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
    for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m, 64);
    s *= a.scale * ks;
    const float now = fmaxf(top, s);
    const float ref = now == -__builtin_inff() ? 0.f : now;  // scores of -inf weigh nothing
    const float keep = expf(top - ref), p = expf(s - ref);
    sum = sum * keep + p;
    for (int e = 0; e < 4; ++e) acc[e] = acc[e] * keep + p * v[e];
    top = now;
  }
  __shared__ float tops[4], sums[4], accs[4][kMaxDim];
  if (lane == 0) tops[wave] = top, sums[wave] = sum;
  for (int e = 0; e < 4; ++e) accs[wave][lane * 4 + e] = acc[e];
  __syncthreads();
  if (wave) return;
  const float all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  float total_sum = 0, out[4] = {0, 0, 0, 0};
  for (int w = 0; w < 4; ++w) {
    const float f = tops[w] == -__builtin_inff() ? 1.f : expf(tops[w] - all);  // then its sum is 0 (or NaN)
    total_sum += f * sums[w];
    for (int e = 0; e < 4; ++e) out[e] += f * accs[w][lane * 4 + e];
  }
  const bool empty = total_sum == 0.f;
  for (int e = 0; e < 4; ++e) out[e] = empty ? 0.f : out[e] / total_sum * vs;
  if (mine) *(Pack<T, 4>*)((T*)a.out + (b * a.q.heads + hq) * pages.dim + lane * 4) = narrow<T, 4>(out);
  if (a.lse && lane == 0) a.lse[b * a.q.heads + hq] = empty ? -__builtin_inff() : all + logf(total_sum);
}

}  // namespace

int64_t attend_workspace(int64_t, int64_t, const KvPages&, int64_t, int64_t) { return 0; }

void attend(const AttendArgs& a, const KvPages& pages, hipStream_t s) {
  if (a.batch == 0 || a.q.heads == 0) return;
  const dim3 grid((unsigned)a.batch, (unsigned)a.q.heads);
  auto kernel = pages.type == kE4M3 ? (a.type == kF16 ? attend_kernel<f16, e4m3> : attend_kernel<bf16, e4m3>)
                                    : (a.type == kF16 ? attend_kernel<f16, f16> : attend_kernel<bf16, bf16>);
  kernel<<<grid, 256, 0, s>>>(a, pages);
  hip_check(hipGetLastError(), "attention");
}

}  // namespace jasper_amd
