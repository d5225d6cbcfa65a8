// kvcache.hpp -- a paged cache of keys and values: its layout, the kernels
// that fill and move it (kvcache.hip) and the attention of one new token that
// reads it (attention.hip).
//
// K and V are each [layers][pages][kv heads][page size][dim]; a sequence's
// token t lies in row t % page_size of page table[t / page_size]. The heads
// come before the rows so that what one work-group reads of a page, a head's
// rows, is one contiguous block (4 KB at 16 rows of 128 fp16 values). Strides
// are the caller's (in values), so a layer of a larger tensor, or pages that
// hold K and V side by side, are read in place; only a row's values are
// contiguous.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jasper_amd {

enum KvType : int32_t { kF16 = 0, kBF16 = 1, kE4M3 = 2 };

struct KvPages {
  char* k = nullptr;
  char* v = nullptr;
  int64_t layer_stride = 0, page_stride = 0, head_stride = 0, row_stride = 0;  // values
  int32_t layers = 1, pages = 0, heads = 0, page = 0, page_shift = 0, dim = 0, type = kF16;
  const float* k_scale = nullptr;  // [heads], a stored value times it is the value; null: 1
  const float* v_scale = nullptr;
};

inline int kv_bytes(int32_t type) { return type == kE4M3 ? 1 : 2; }

// One tensor of rows [n][heads][dim], contiguous in its last dimension.
struct HeadRows {
  const void* p = nullptr;
  int64_t stride = 0, head_stride = 0;  // values
  int32_t heads = 0;
};

// q and k (heads 0: absent) with the first 2 * half values of every head
// turned by the angles of their positions' table rows, to contiguous q_out,
// k_out. back: by the opposite angles (the gradient). Rows whose position is
// outside the table get NaN.
struct RotaryArgs {
  HeadRows q, k;
  const void* positions = nullptr;
  bool pos64 = true, interleaved = false, back = false;
  const float* cos = nullptr;
  const float* sin = nullptr;
  int64_t n = 0, table_rows = 0;
  int32_t dim = 0, half = 0, type = kF16;
};
void rotary(const RotaryArgs& a, void* q_out, void* k_out, hipStream_t s);

// The same for the tokens of a serving step: q to q_out, k rotated and v as
// it is to row slots[i] % page_size of page slots[i] / page_size. A slot
// outside the cache is skipped (its q is rotated all the same). half = 0:
// nothing is rotated.
void append_tokens(const RotaryArgs& a, const HeadRows& v, const void* slots, bool slots64, const KvPages& pages,
                   void* q_out, hipStream_t s);

// Pages src[i] to dst[i], K and V of every layer; with tables (entries of any
// number of sequences, as one list), entries equal to src[i] become dst[i].
// No page may be both a source and a destination. Pairs with an id outside
// the cache are skipped.
void copy_pages(const KvPages& pages, const int32_t* src, const int32_t* dst, int64_t n, int32_t* tables,
                int64_t table_entries, hipStream_t s);

// Attention of one new token per sequence. lists 0: over the last `last`
// tokens of the cache (all when last < 0). With ids [batch][lists][count]:
// over the first `first`, the last `last` and those ids in between them.
struct AttendArgs {
  HeadRows q;  // stride: between sequences
  int32_t type = kF16;
  const int32_t* tables = nullptr;
  int64_t table_stride = 0;
  int32_t table_width = 0;
  const int32_t* lens = nullptr;
  int64_t batch = 0, max_len = 0;
  float scale = 0;
  const int32_t* ids = nullptr;
  int32_t lists = 0, count = 0;
  int64_t first = 0, last = -1;
  void* out = nullptr;    // [batch][heads][dim]
  float* lse = nullptr;   // [batch][heads] or null
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};
// Scratch bytes of a call that reads up to max_tokens tokens per head (lists
// 0: no ids).
int64_t attend_workspace(int64_t batch, int64_t q_heads, const KvPages& pages, int64_t max_tokens, int64_t lists);
void attend(const AttendArgs& a, const KvPages& pages, hipStream_t s);

}  // namespace jasper_amd
