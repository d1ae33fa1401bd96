// The paged cache's bookkeeping (pages.cu) and a batch's view of it, as the attention over its pages (paged_attn.cu) uses them.
#pragma once
#include <exception>
#include <new>
#include <vector>

#include "tc_common.cuh"

namespace infllm {

struct PageSeq {
  bool open = false;
  uint32_t generation = 0;  // counts the sequences that had this number
  uint64_t changes = 0;     // of its tokens: some added, or taken away
  int64_t length = 0, position = 0;
  std::vector<int32_t> pages;
};

// The pages that no sequence has: a bit each, taken lowest first.  No page below word `first_` is free.
class FreePages {
 public:
  void fill(int32_t n) {
    words_.assign((size_t)(n + 63) / 64, ~0ull);
    if (n % 64) words_.back() = (1ull << (n % 64)) - 1;
    first_ = 0, count_ = n;
  }
  int32_t count() const { return count_; }
  int32_t take() {  // (of some)
    while (!words_[first_]) ++first_;
    const int bit = __builtin_ctzll(words_[first_]);
    words_[first_] &= words_[first_] - 1;
    --count_;
    return (int32_t)(first_ * 64) + bit;
  }
  void give(int32_t page) {
    const size_t at = (size_t)page / 64;
    words_[at] |= 1ull << (page % 64);
    if (at < first_) first_ = at;
    ++count_;
  }

 private:
  std::vector<uint64_t> words_;
  size_t first_ = 0;
  int32_t count_ = 0;
};

// One launch's worth of changes: rows of the table that are copied, entries that are set, tokens that are moved.
struct PageItem {
  int32_t a, b, c, d;
};

// A batch's tokens as the kernels get them.
struct BatchSeq {
  int32_t row;       // of the table
  int32_t length;    // tokens, the newest included
  int32_t count;     // of them the newest that the call is about
  int32_t position;  // of the first of those, for the rotary embedding
};

// the current device for a call's duration
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (device >= 0 && cudaGetDevice(&before_) == cudaSuccess && before_ != device) ok_ = cudaSetDevice(device) == cudaSuccess;
    else before_ = -1;
  }
  ~DeviceScope() {
    if (before_ >= 0) cudaSetDevice(before_);
  }
  bool ok() const { return ok_; }

 private:
  int before_ = -1;
  bool ok_ = true;
};

// nothing is thrown across the C boundary
template <typename F>
int guarded(const char* what, F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(INFLLM_E_NOMEM, "%s: no host memory", what);
  } catch (const std::exception& e) {
    return fail(INFLLM_E_NOMEM, "%s: %s", what, e.what());
  }
}

}  // namespace infllm

struct infllm_pages {
  infllm_pages_config cfg;
  std::vector<infllm::PageSeq> seqs;
  std::vector<int32_t> uses;  // sequences that have a page
  infllm::FreePages free_pages;
  uint64_t change = 0;   // any change of what sequences hold
  uint64_t reshape = 0;  // of which pages sequences share, but for forks
  std::vector<infllm::PageItem> rows, edits, moves;  // of the call that is being made (pages.cu)
  std::vector<int32_t> to_pages;
  CUtensorMap map;       // of all pages (paged_tc.cu)
  int32_t n_sm = 148;
  int32_t* lost = nullptr;  // pinned: written by a block whose wait ran out (code, wait, block), read by the next calls

  ~infllm_pages();
  int32_t pages_of(int64_t tokens) const { return (int32_t)((tokens + cfg.page_size - 1) / cfg.page_size); }
};

struct infllm_page_batch {
  infllm_pages* cache;
  std::vector<int32_t> seqs;
  std::vector<uint32_t> generation;
  std::vector<int32_t> count;  // newest tokens of each sequence that calls are about
  std::vector<uint64_t> as_of;  // each sequence's `changes` when they were set
  int32_t most = 0;            // the largest of them: the tokens of a call's tensors
  // the order of the sequences by their pages, and how many pages each shares with the one before: as of `reshape`
  uint64_t order_of = ~0ull;
  std::vector<int32_t> order, common;
  // the plan of the attention (paged_attn.cu), as of `change` and for n_heads
  uint64_t plan_of = ~0ull;
  int32_t plan_heads = 0;
  bool upload = false;  // it is not on the device yet
  std::vector<int32_t> plan;
  int32_t n_row_units = 0, n_ctas = 0;
  int32_t n_beside = 0;   // units of few rows that go to the blocks of many, the first; the others:
  int32_t most_rows = 0;  // of a unit
  bool join = false;
  int64_t part_rows = 0;
  int64_t off_unit = 0, off_tile_unit = 0, off_cta = 0, off_seq = 0, off_path = 0, off_span = 0, off_node_seq = 0;  // sections of the plan
};

namespace infllm {
int batch_alive(const infllm_page_batch* b, const char* what);
int check_lost(infllm_pages* p, cudaStream_t s);  // paged_attn.cu
int pages_encode_map(infllm_pages* p);  // paged_tc.cu
}  // namespace infllm
