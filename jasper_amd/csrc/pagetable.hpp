// pagetable.hpp -- which pages the sequences of a paged cache have, kept on the
// GPU (pagetable.hip): sequences grow, are cut back and forked by kernels, so
// that a whole step can be captured in a graph.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jasper_amd {

// tables [sequences][width]: a sequence's pages in order, -1 behind them; lens
// [sequences]: its tokens; refs [pages]: how many sequences have a page; free:
// a bit for each page, the lowest first, set where refs is 0.
struct PageState {
  int32_t* tables = nullptr;
  int32_t* lens = nullptr;
  int32_t* refs = nullptr;
  uint32_t* free = nullptr;
  int32_t sequences = 0, width = 0, pages = 0, page_shift = 0;
};

// counts[i] more tokens for sequence seqs[i], i < n. Outputs as in the header.
struct ExtendArgs {
  const int32_t* seqs = nullptr;
  const int32_t* counts = nullptr;
  int64_t n = 0, n_tokens = 0;
  int32_t width = 0;  // of step_tables
  int64_t* positions = nullptr;
  int64_t* slots = nullptr;
  int32_t* starts = nullptr;
  int32_t* step_tables = nullptr;
  int32_t* step_lens = nullptr;
  int32_t* src = nullptr;
  int32_t* dst = nullptr;
  int32_t* missing = nullptr;
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};
int64_t extend_workspace(int64_t n, int64_t pages);
void extend_tables(const PageState& state, const ExtendArgs& a, hipStream_t s);

// The sequences cut back to to[i] tokens; pages that nobody has any more are free.
void truncate_tables(const PageState& state, const int32_t* seqs, const int32_t* to, int64_t n, hipStream_t s);

// Empty sequences into[i] get the tokens of seqs[i], on the same pages.
void fork_tables(const PageState& state, const int32_t* seqs, const int32_t* into, int64_t n, hipStream_t s);

// Neighbours of a batch with the same first pages: groups [batch + 1], shared [batch].
int64_t prefixes_workspace(int64_t batch);
void shared_prefixes(const int32_t* tables, int64_t stride, int64_t width, const int32_t* lens, int64_t batch,
                     int32_t page_shift, int64_t least, int32_t* groups, int32_t* shared, void* workspace,
                     int64_t workspace_bytes, hipStream_t s);

}  // namespace jasper_amd
