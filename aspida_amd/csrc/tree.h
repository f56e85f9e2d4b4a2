// tree.h -- trees of drafted tokens: masks and positions, and the greedy
// choice along a tree.
//
// A sequence's rows are a tree: row 0 is the last token that is sure, every
// other row a drafted token behind its parent, an earlier row.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace kq {

constexpr int TREE_MAX_WORDS = 128;                  // of a mask row
constexpr int TREE_MAX_ROWS = 32 * TREE_MAX_WORDS;   // of a sequence

struct TreeRows {
  const int *parent, *row_start, *kv_len;
  int n_rows, n_seq;
};
// mask [n_rows][words], bit j of a row: the row j of its sequence is an
// ancestor or itself; pos: kv_len - rows + depth.  Either may be null.
hipError_t launch_tree(const TreeRows& t, int* pos, uint32_t* mask, int words, hipStream_t s);

struct TreeAccept {
  const void* logits;
  long long stride;
  int vocab;
  const int* token;
  int *path, *count, *next, *new_len;
  void* work;
};
size_t tree_accept_work_bytes(int n_rows, int vocab);
hipError_t launch_tree_accept(int type, const TreeRows& t, const TreeAccept& a, hipStream_t s);

}  // namespace kq
