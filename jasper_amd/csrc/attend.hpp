// attend.hpp -- one wave over a stream of the cache's tokens under up to 16
// query rows, on the matrix cores: what the attention kernels (attention.hip,
// shared.hip) are made of.
#pragma once

#include "kvtypes.hpp"

#include <type_traits>

namespace jasper_amd {
namespace attention {

constexpr int kTile = 32;    // tokens a wave takes at once
constexpr int kHeads = 16;   // query heads of a matrix instruction
constexpr int kStart = 2;    // what beginning a stream costs a wave, in tiles
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  const char* q;
  int64_t q_stride, q_head;
  const char *k, *v;
  int64_t page_stride, head_stride, row_stride;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* ids;
  const float *k_scale, *v_scale;
  char* out;
  float* lse;
  float* parts;
  int2* ends;
  float scale;  // times log2(e)
  int batch, heads, q_heads, lists, group, count;
  int head_tiles, side;  // 16s of a list's query heads, and how many of them share a work-group
  int part_heads;
  int page_shift, pages, dim;
  int limit, first, last;  // tokens; last: -1 for all
};

typedef uintx4 Frag;  // 8 values of 16 bits

template <typename T>
__device__ __forceinline__ floatx4 mfma(Frag a, Frag b, floatx4 c) {
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
  if constexpr (std::is_same_v<T, f16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef T pair __attribute__((ext_vector_type(2)));
  const pair p = {(T)a, (T)b};
  return __builtin_bit_cast(uint32_t, p);
}

template <typename T>
__device__ __forceinline__ floatx2 unpack2(uint32_t w) {
  if constexpr (std::is_same_v<T, f16>) {
    typedef T pair __attribute__((ext_vector_type(2)));
    const pair p = __builtin_bit_cast(pair, w);
    return floatx2{(float)p.x, (float)p.y};
  } else {
    return floatx2{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xFFFF0000u)};
  }
}

// Two of a word's four e4m3 bytes as two values of T (exact in both types).
template <typename T>
__device__ __forceinline__ uint32_t from_e4m3(uint32_t w, bool high) {
  if constexpr (std::is_same_v<T, f16>)
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  else
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
}

// Rows are read once, past the caches (four sequences of 131k tokens: 175 us,
// 191 with ordinary loads). Not where a row is no whole number of 128-byte
// lines: neighbours share lines, and 96 dims took 79 us instead of 76.
template <bool STREAM, typename W>
__device__ __forceinline__ W load(const W* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}

// What a sequence has its queries read: the tokens [begin, end), counted from
// base in tiles; of a list's places [0, end) the first `first` are tokens,
// then come the tokens from `last` on, then the ids.
struct Span {
  int base, begin, end, tiles, cost;  // base: begin rounded down to whole groups of 8 rows
  int first, last;
};

template <bool LISTED>
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  Span s;
  const int len = min(max(p.lens[b], 0), p.limit);
  if (LISTED) {
    s.first = min(p.first, len);
    s.last = max(len - p.last, s.first);
    s.base = s.begin = 0;
    s.end = s.first + (len - s.last) + p.count;
  } else {
    s.begin = p.last >= 0 && len > p.last ? len - p.last : 0;
    s.base = s.begin & ~7;
    s.end = len;
  }
  s.tiles = max(1, (s.end - s.base + kTile - 1) / kTile);  // a sequence of no tokens has its zeros written
  s.cost = kStart + s.tiles;
  return s;
}

// How the work of all sequences and streams is shared out. A stream of n
// tiles counts kStart + n units, as a wave that begins it first waits for its
// queries and rows: of sequences with 17 to 8192 tokens, waves with equal
// tiles took 71 us, the slowest ones eight short streams each. The first
// `more` of `waves` waves have each + 1 units, the others each.
struct Share {
  int each, more, waves;
  __device__ int begin(int w) const { return each * w + min(w, more); }
  __device__ int owner(int unit) const {
    const int longer = (each + 1) * more;
    return unit < longer ? unit / (each + 1) : more + (unit - longer) / each;
  }
};

// A stream: the tokens of one sequence under up to 16 query heads of a list.
struct Stream {
  int b, list, heads, q_head, kv_head;
};

__device__ __forceinline__ Stream stream_of(const Params& p, int b, int list, int head_tile) {
  const int head0 = head_tile * kHeads;
  return {b, list, min(kHeads, p.group - head0), list * p.group + head0, list * p.heads / p.lists};
}

// A wave's sums over some tiles: o (of V, by lane as above) and `sum` (of the
// weights) are 2^-ref times what they stand for.
template <int DT>
struct Sums {
  floatx4 o[DT / 16];
  float ref, sum;
};

// The dims of o[j][r].
template <bool F8, int DT>
__device__ __forceinline__ int dim_of(int g, int j, int r) {
  constexpr int BD = DT / 16 * (F8 ? 1 : 2) > 16 ? 8 : DT / 16;
  return j / BD * 16 * BD + (4 * g + r) * BD + j % BD;
}

// LDS that only this wave reads and writes: kept in order, not waited for.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The query of a lane's head.
__device__ __forceinline__ const char* query_of(const Params& p, const Stream& at, int i) {
  return p.q + (at.b * p.q_stride + (at.q_head + i) * p.q_head) * 2;
}

// One wave over tiles [c, c1) of a stream; q_row: the lane's query, of lanes
// below at.heads (of 16); rows: STAGE offsets in LDS.
//
// S = K Q^T and O^T = V^T P^T on 16x16x32 instructions, all in registers. With
// g = lane / 16, i = lane % 16 and 8 tokens to a group, a tile of 32 tokens is
//  K  two operands' rows i: token 8 (i / 4) + i % 4 (+ 4 in the second); so
//  S  comes out with lane (g, i) holding head i's scores of group g's eight
//     tokens, which is where P has to be as the operand of the second product:
//     nothing crosses lanes.
//  V  lane (g, i) loads VD dims of group g's eight tokens, in blocks of up to
//     16 bytes of which 16 lanes read a contiguous run: dims BD i on, and 16
//     BD further in each next block. The 8 x VD values are turned with byte
//     permutes into VD operands, product j giving the j-th dims of all lanes.
//  O  lane (g, i): head i, of dims that lane 4 g + r loads the j-th in o[j][r].
// Heads past the group's are zero queries: the loads bound the kernel, not the
// products (of fp16 rows of 128 values 24 instructions of 16 cycles for the 16
// KB of a tile; weights of one term would spare 8 of them, and 1 us of 71).
template <typename T, bool F8, int DT, bool LISTED, bool FULL, int STAGE>
__device__ __forceinline__ Sums<DT> attend_tiles(const Params& p, const Span& sp, const Stream& at, const char* q_row,
                                                 int c, int c1, int64_t* rows) {
  constexpr int VD = DT / 16, KS = DT / 32, ES = F8 ? 1 : 2;
  constexpr int BD = VD * ES > 16 ? 16 / ES : VD;  // dims of a lane that lie together
  typedef std::conditional_t<F8, f16, T> PT;  // e4m3 values are exact in fp16, where weights keep more bits
  // The reference is moved once a score is 2^3 above the one it was set for.
  // fp16 weights are 2^12 larger, so that those far below the largest are not
  // lost; bf16's are at most 1, as V may reach fp32's end.
  constexpr float kLag = 3.f, kTop = std::is_same_v<PT, f16> ? 12.f : -kLag;
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const char* kb = p.k + at.kv_head * p.head_stride * ES;
  const char* vb = p.v + at.kv_head * p.head_stride * ES;
  const float cs = p.scale * (p.k_scale ? p.k_scale[at.kv_head] : 1.f);

  Frag q[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d = F8 ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
    q[s] = Frag{0, 0, 0, 0};
    if (i < at.heads && (FULL || d < p.dim)) q[s] = *(const Frag*)(q_row + d * 2);
  }
  Sums<DT> out;
  floatx4 (&o)[VD] = out.o;
#pragma unroll
  for (int j = 0; j < VD; ++j) o[j] = floatx4{0, 0, 0, 0};
  float ref = -__builtin_inff(), use = 0.f, sum = 0.f;

  constexpr int kStageTiles = STAGE / (LISTED ? kTile : kTile / 8);
  const int n_all = sp.end > sp.base ? c1 : c;  // no tokens, no tiles
  for (int c0 = c; c0 < n_all; c0 += kStageTiles) {
    const int n_tiles = min(n_all - c0, kStageTiles);
    // offsets of the rows: one per token of a list, one per 8 tokens else
    wave_sync();
    for (int e = lane; e < n_tiles * (LISTED ? kTile : kTile / 8); e += 64) {
      int t;
      int64_t off = -1;
      bool known;
      if (LISTED) {
        const int place = c0 * kTile + e, always = sp.end - p.count;
        known = place < sp.end;
        t = place < sp.first ? place : sp.last + (place - sp.first);
        if (known && place >= always) {
          t = p.ids[((int64_t)at.b * p.lists + at.list) * p.count + (place - always)];
          known = t >= sp.first && t < sp.last;
        }
      } else {
        t = sp.base + c0 * kTile + 8 * e;
        known = t < sp.end;
      }
      if (known) {
        const int32_t page = p.tables[at.b * p.table_stride + (t >> p.page_shift)];
        if (page >= 0 && page < p.pages)
          off = (page * p.page_stride + (t & ((1 << p.page_shift) - 1)) * p.row_stride) * ES;
      }
      rows[e] = off;
    }
    wave_sync();

    Frag kf[2][KS];
    auto load_k = [&](int tile) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int tok = 8 * (i >> 2) + (i & 3) + 4 * r;
        int64_t off = LISTED ? rows[tile * kTile + tok] : rows[tile * (kTile / 8) + (i >> 2)];
        off = off < 0 ? 0 : off;
        if (!LISTED) off += ((i & 3) + 4 * r) * p.row_stride * ES;
        const char* row = kb + off;
        if constexpr (F8) {
#pragma unroll
          for (int s = 0; s < KS; s += 2) {
            const int d = 32 * s + 16 * g;
            const bool in = FULL || d < p.dim;
            uintx4 w = load<FULL>((const uintx4*)(row + (in ? d : 0)));
            if (!in) w = uintx4{0, 0, 0, 0};
            kf[r][s] = Frag{w.x, w.y, 0, 0};
            kf[r][s + 1] = Frag{w.z, w.w, 0, 0};
          }
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int d = 32 * s + 8 * g;
            const bool in = FULL || d < p.dim;
            uintx4 w = load<FULL>((const uintx4*)(row + (in ? d : 0) * 2));
            if (!in) w = uintx4{0, 0, 0, 0};
            kf[r][s] = w;
          }
        }
      }
    };
    constexpr int VW = VD * ES / 4;  // words of V per token and lane
    // a chunk of V past the end of a row is the row's first instead: those dims are never stored
    const auto v_at = [&](int w) {
      const int d = w / 4 * 16 * BD + i * BD;
      return FULL || d < p.dim ? d * ES : 0;
    };

    // one tile, with the next one's keys on their way while its values are
    auto step = [&](int tile, auto more) {
      uint32_t vw[8][VW];
      uint32_t valid = 0;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        int64_t off = LISTED ? rows[tile * kTile + 8 * g + t] : rows[tile * (kTile / 8) + g];
        bool in = off >= 0;
        if (!LISTED) {
          const int tok = sp.base + (c0 + tile) * kTile + 8 * g + t;
          in = in && tok >= sp.begin && tok < sp.end;
        }
        valid |= in ? 1u << t : 0u;
        off = off < 0 ? 0 : off;
        if (!LISTED) off += t * p.row_stride * ES;
        const char* row = vb + off;
        if constexpr (VW >= 4) {
#pragma unroll
          for (int w = 0; w < VW; w += 4) {
            const uintx4 y = load<FULL>((const uintx4*)(row + v_at(w)));
            vw[t][w] = y.x, vw[t][w + 1] = y.y, vw[t][w + 2] = y.z, vw[t][w + 3] = y.w;
          }
        } else if constexpr (VW == 2) {
          const uintx2 y = load<FULL>((const uintx2*)(row + v_at(0)));
          vw[t][0] = y.x, vw[t][1] = y.y;
        } else {
          vw[t][0] = load<FULL>((const uint32_t*)(row + v_at(0)));
        }
      }
      floatx4 s[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        s[r] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < KS; ++e) {
          Frag a = kf[r][e];
          if constexpr (F8)
            a = Frag{from_e4m3<T>(a.x, false), from_e4m3<T>(a.x, true), from_e4m3<T>(a.y, false), from_e4m3<T>(a.y, true)};
          s[r] = mfma<T>(a, q[e], s[r]);
        }
      }
      if constexpr (more.value) load_k(tile + 1);
      float z[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) z[t] = s[t >> 2][t & 3] * cs;
      if (!__all(valid == 0xFFu)) {
        // what stands in masked rows may be anything: neither its scores nor its values are used
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const bool in = valid >> t & 1;
          z[t] = in ? z[t] : -__builtin_inff();
#pragma unroll
          for (int w = 0; w < VW; ++w) vw[t][w] = in ? vw[t][w] : 0u;
        }
      }
      float top = z[0];
#pragma unroll
      for (int t = 1; t < 8; ++t) top = fmaxf(top, z[t]);
      if (__any(top > ref + (kTop + kLag))) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float now = fmaxf(ref, top - kTop);
        const float to = now == -__builtin_inff() ? 0.f : now;
        const float keep = __builtin_amdgcn_exp2f(ref - to);
        sum *= keep;
#pragma unroll
        for (int j = 0; j < VD; ++j) o[j] *= keep;
        ref = now, use = to;
      }
      // the weights in two terms of their type, so that their rounding adds
      // nothing to the output's own
      Frag hi, lo;
#pragma unroll
      for (int t = 0; t < 8; t += 2) {
        const float a = __builtin_amdgcn_exp2f(z[t] - use), bb = __builtin_amdgcn_exp2f(z[t + 1] - use);
        sum += a + bb;
        hi[t / 2] = pack2<PT>(a, bb);
        const floatx2 back = unpack2<PT>(hi[t / 2]);
        lo[t / 2] = pack2<PT>(a - back.x, bb - back.y);
      }
      // turn V: word w of tokens t, t + 1 holds dims 2w, 2w + 1 (bytes: 4)
      constexpr int kPer = 4 / ES;
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        Frag f[kPer];
#pragma unroll
        for (int t = 0; t < 8; t += 2) {
          if constexpr (F8) {
            const uint32_t even = __builtin_amdgcn_perm(vw[t + 1][w], vw[t][w], 0x05010400u);
            const uint32_t odd = __builtin_amdgcn_perm(vw[t + 1][w], vw[t][w], 0x07030602u);
            f[0][t / 2] = from_e4m3<PT>(even, false), f[1][t / 2] = from_e4m3<PT>(even, true);
            f[2][t / 2] = from_e4m3<PT>(odd, false), f[3][t / 2] = from_e4m3<PT>(odd, true);
          } else {
            f[0][t / 2] = __builtin_amdgcn_perm(vw[t + 1][w], vw[t][w], 0x05040100u);
            f[1][t / 2] = __builtin_amdgcn_perm(vw[t + 1][w], vw[t][w], 0x07060302u);
          }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          o[kPer * w + j] = mfma<PT>(f[j], hi, o[kPer * w + j]);
          o[kPer * w + j] = mfma<PT>(f[j], lo, o[kPer * w + j]);
        }
      }
    };
    load_k(0);
    for (int tile = 0; tile + 1 < n_tiles; ++tile) step(tile, std::true_type{});
    step(n_tiles - 1, std::false_type{});
  }

  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  out.ref = ref, out.sum = sum;
  return out;
}

}  // namespace attention
}  // namespace jasper_amd
