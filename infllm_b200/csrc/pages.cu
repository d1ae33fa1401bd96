// A paged key/value cache: sequences of tokens in pages of a pool, several of which may share pages (the continuations of
// one prompt).  Which pages a sequence has is known on the host, exactly and at once: what does not fit is refused before
// anything changes, and a call's grid follows from sizes that the host has.  The device has a copy of the page table.
//
// Layout: a page of one layer holds its tokens' keys, (n_kv_heads, page_size, head_dim), and in another plane their values;
// a page's plane is one stretch of memory, and so are the rows of one head.  Rows of a page that are in use are never
// written again while two sequences share it: a sequence has its last page, where that is not full, to itself (fork copies
// it; where truncation left it shared, it is copied before the next token is written).
#include <algorithm>
#include <cstring>
#include <mutex>

#include "pages.cuh"

namespace infllm {

// ---------------------------------------------------------------------------------------------------------- changes
// One kernel makes all changes of a call: items [0, n_rows) copy a row of the table (a: from row, b: to row, c: entries),
// the next n_edits set entries (a: index, b: page, and c, d another one, index -1: none), the next n_moves move tokens in all
// layers, keys and values (a: from page, b: the first of the pages to move them to, c: from place | to place << 16, d: tokens |
// pages << 16); those pages' numbers are behind them, four to an item.
// Pages that are written were free before the call, and rows that are written belong to sequences that are not read from, so
// that the order of the blocks does not matter.  It is bound by the bytes of the tokens, read once and written as often as there
// are pages for them: half of two 65536-token sequences of four layers (2.1 GB) in 326 us, 6.6 TB/s; the last page of a sequence
// for 64 forks in eight layers (268 MB written) in 47.
constexpr int kMoveThreads = 256;
constexpr int kMoveAhead = 8;  // 16-byte loads of a thread in flight
constexpr int kChunk = 256;    // 16-byte pieces that a warp takes at once
constexpr int kMostTo = 256;   // pages of a move

template <int kItems>
struct PageChanges {
  const char* from;  // the pools that tokens are moved from and to, of from_pages and to_pages pages
  char* to;
  int32_t* table;
  int32_t n_rows, n_edits, n_moves, max_pages;
  int32_t parts, shares;  // blocks of a move: parts of its tokens by shares of the pages that they go to
  int32_t planes, from_pages, to_pages, n_kv, page, dim16;  // dim16: 16-byte pieces of a row
  PageItem item[kItems];
};

template <int kItems>
__global__ void __launch_bounds__(kMoveThreads) page_change_kernel(const __grid_constant__ PageChanges<kItems> P) {
  int b = blockIdx.x;
  if (b < P.n_rows) {
    const PageItem it = P.item[b];
    const int32_t* from = P.table + (int64_t)it.a * P.max_pages;
    int32_t* to = P.table + (int64_t)it.b * P.max_pages;
    for (int i = threadIdx.x; i < it.c; i += kMoveThreads) to[i] = from[i];
    return;
  }
  b -= P.n_rows;
  if (P.n_edits > 0 && b-- == 0) {
    for (int i = threadIdx.x; i < P.n_edits; i += kMoveThreads) {
      const PageItem it = P.item[P.n_rows + i];
      P.table[it.a] = it.b;
      if (it.c >= 0) P.table[it.c] = it.d;
    }
    return;
  }
  const PageItem it = P.item[P.n_rows + P.n_edits + b / (P.parts * P.shares)];
  const int32_t* pages = reinterpret_cast<const int32_t*>(P.item + P.n_rows + P.n_edits + P.n_moves) + it.b;
  const int part = b % P.parts, to0 = b / P.parts % P.shares, n_to = it.d >> 16;
  const int from = it.c & 0xffff, to = it.c >> 16;
  // Rows of a head in a plane are one stretch on both sides; a warp takes up to 4 KB of one.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int strip = (it.d & 0xffff) * P.dim16, chunks = (strip + kChunk - 1) / kChunk, units = P.planes * P.n_kv * chunks;
  const int u1 = (int)((int64_t)units * (part + 1) / P.parts);
  const int head = P.page * P.dim16;  // pieces of a head's rows of a page
  const int64_t page16 = (int64_t)P.n_kv * head;
  for (int u = (int)((int64_t)units * part / P.parts) + warp; u < u1; u += kMoveThreads / 32) {
    const int s = u / chunks, plane = s / P.n_kv, h = s - plane * P.n_kv, i0 = (u - s * chunks) * kChunk, i1 = min(strip, i0 + kChunk);
    const uint4* src = reinterpret_cast<const uint4*>(P.from) + ((int64_t)plane * P.from_pages + it.a) * page16 + h * head + from * P.dim16;
    uint4* dst = reinterpret_cast<uint4*>(P.to) + (int64_t)plane * P.to_pages * page16 + h * head + to * P.dim16;
    for (int i = i0 + lane; i < i1; i += 32 * kMoveAhead) {
      uint4 v[kMoveAhead];
#pragma unroll
      for (int k = 0; k < kMoveAhead; ++k)
        if (i + k * 32 < i1) v[k] = src[i + k * 32];
#pragma unroll 1
      for (int x = to0; x < n_to; x += P.shares) {
        uint4* d = dst + pages[x] * page16;
#pragma unroll
        for (int k = 0; k < kMoveAhead; ++k)
          if (i + k * 32 < i1) d[i + k * 32] = v[k];
      }
    }
  }
}

// Items of one launch: a stretch of each list.
struct ChangeSpan {
  size_t r0, r1, e0, e1, m0, m1;
};

template <int kItems>
static int launch_changes(infllm_pages* p, const infllm_pages* from, const ChangeSpan& c, cudaStream_t s) {
  const infllm_pages_config& g = p->cfg;
  PageChanges<kItems> P;
  P.from = (const char*)from->cfg.d_pages, P.to = (char*)g.d_pages;
  P.table = g.d_table;
  P.n_rows = (int)(c.r1 - c.r0), P.n_edits = (int)(c.e1 - c.e0), P.n_moves = (int)(c.m1 - c.m0), P.max_pages = g.max_pages;
  P.planes = 2 * g.n_layers, P.from_pages = from->cfg.n_pages, P.to_pages = g.n_pages;
  P.n_kv = g.n_kv_heads, P.page = g.page_size, P.dim16 = g.head_dim / 8;
  PageItem* at = P.item;
  at = std::copy(p->rows.begin() + c.r0, p->rows.begin() + c.r1, at);
  at = std::copy(p->edits.begin() + c.e0, p->edits.begin() + c.e1, at);
  int32_t most = 0, most_to = 1;
  if (c.m1 > c.m0) {
    const int32_t first = p->moves[c.m0].b, last = p->moves[c.m1 - 1].b + (p->moves[c.m1 - 1].d >> 16);
    for (size_t i = c.m0; i < c.m1; ++i, ++at) {
      *at = p->moves[i];
      at->b -= first;
      most = std::max(most, at->d & 0xffff), most_to = std::max(most_to, at->d >> 16);
    }
    std::copy(p->to_pages.begin() + first, p->to_pages.begin() + last, reinterpret_cast<int32_t*>(at));
  }
  // a piece of work for every warp of a block, or two where there are many; and the pages of a move shared out until there are sixteen
  // blocks per SM (64 forks of a page in eight layers, 268 MB written: 67 us by blocks that have all 64 pages, 47 so)
  const int64_t units = (int64_t)P.planes * P.n_kv * ceil_div(most * P.dim16, kChunk), warps = kMoveThreads / 32, enough = (int64_t)p->n_sm * 16;
  P.parts = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(units, P.n_moves * units > 2 * enough * warps ? 2 * warps : warps), 65535));
  P.shares = (int)std::max<int64_t>(1, std::min<int64_t>(most_to, enough / std::max<int64_t>(1, (int64_t)P.n_moves * P.parts)));
  const int64_t blocks = P.n_rows + (P.n_edits > 0) + (int64_t)P.n_moves * P.parts * P.shares;
  page_change_kernel<kItems><<<(unsigned)blocks, kMoveThreads, 0, s>>>(P);
  INFLLM_LAUNCH_OK("page_change_kernel");
  return INFLLM_OK;
}

// makes the changes that a call has listed; tokens are moved from the pages of `from`
static int flush(infllm_pages* p, const infllm_pages* from, cudaStream_t s) {
  // items of 16 bytes: a kernel's arguments, of 1, 4 and 16 KB (a launch costs about 0.3 us more per KB)
  constexpr size_t kSmall = 56, kMiddle = 250, kLarge = 1000;
  static_assert(kLarge > 2 + kMostTo / 4, "");
  int rc = INFLLM_OK;
  if (p->cfg.device >= 0) {
    ChangeSpan c{0, 0, 0, 0, 0, 0};
    while (rc == INFLLM_OK && (c.r1 < p->rows.size() || c.e1 < p->edits.size() || c.m1 < p->moves.size())) {
      size_t used = 0;
      c.r0 = c.r1, c.e0 = c.e1, c.m0 = c.m1;
      c.r1 = std::min(p->rows.size(), c.r0 + kLarge), used += c.r1 - c.r0;
      c.e1 = std::min(p->edits.size(), c.e0 + kLarge - used), used += c.e1 - c.e0;
      size_t to = 0;  // pages of the moves
      while (c.m1 < p->moves.size()) {
        const size_t more = to + (size_t)(p->moves[c.m1].d >> 16);
        if (used + (c.m1 - c.m0 + 1) + (more + 3) / 4 > kLarge) break;
        to = more, ++c.m1;
      }
      used += c.m1 - c.m0 + (to + 3) / 4;
      rc = used <= kSmall ? launch_changes<kSmall>(p, from, c, s) : used <= kMiddle ? launch_changes<kMiddle>(p, from, c, s) : launch_changes<kLarge>(p, from, c, s);
    }
  }
  p->rows.clear();
  p->edits.clear();
  p->moves.clear();
  p->to_pages.clear();
  return rc;
}

// ------------------------------------------------------------------------------------------------------ bookkeeping
static int check_seqs(const infllm_pages* p, const int32_t* seqs, int n, const char* what) {
  if (!p || n < 0 || (n > 0 && !seqs)) return fail(INFLLM_E_BADARG, "%s: null pointer or a negative count", what);
  for (int i = 0; i < n; ++i)
    if (seqs[i] < 0 || seqs[i] >= (int)p->seqs.size() || !p->seqs[seqs[i]].open)
      return fail(INFLLM_E_BADARG, "%s: %d is not a sequence of this cache", what, seqs[i]);
  return INFLLM_OK;
}

static int check_once(const infllm_pages* p, const int32_t* seqs, int n, const char* what) {
  INFLLM_TRY(check_seqs(p, seqs, n, what));
  std::vector<char> seen(p->seqs.size(), 0);
  for (int i = 0; i < n; ++i)
    if (seen[seqs[i]]++) return fail(INFLLM_E_BADARG, "%s: sequence %d is named twice", what, seqs[i]);
  return INFLLM_OK;
}

static int32_t take_page(infllm_pages* p) {
  const int32_t page = p->free_pages.take();
  p->uses[page] = 1;
  return page;
}

static void drop_page(infllm_pages* p, int32_t page) {
  if (--p->uses[page] == 0) p->free_pages.give(page);
}

static void set_entry(infllm_pages* p, int32_t row, size_t at, int32_t page) {
  const int32_t index = row * p->cfg.max_pages + (int32_t)at;
  if (!p->edits.empty() && p->edits.back().c < 0) p->edits.back().c = index, p->edits.back().d = page;
  else p->edits.push_back({index, page, -1, 0});
}

// (a move of the same tokens as the last one's is the last one, to another page too)
static void move_tokens(infllm_pages* p, int32_t from, int32_t from_at, int32_t to, int32_t to_at, int32_t n) {
  const int32_t at = from_at | to_at << 16;
  p->to_pages.push_back(to);
  if (!p->moves.empty()) {
    PageItem& m = p->moves.back();
    if (m.a == from && m.c == at && (m.d & 0xffff) == n && (m.d >> 16) < kMostTo) {
      m.d += 1 << 16;
      return;
    }
  }
  p->moves.push_back({from, (int32_t)p->to_pages.size() - 1, at, n | 1 << 16});
}

static int need_pages(const infllm_pages* p, int64_t n, const char* what) {
  if (n > p->free_pages.count())
    return fail(INFLLM_E_CAPACITY, "%s: %lld pages are needed, %d of %d are free", what, (long long)n, p->free_pages.count(), p->cfg.n_pages);
  return INFLLM_OK;
}

// (in a capture the changes would not be made now, and made again with every replay)
static int need_stream(const infllm_pages* p, void* stream, const char* what) {
  if (p->cfg.device < 0) return INFLLM_OK;
  cudaStreamCaptureStatus capture;
  INFLLM_CUDA_OK(cudaStreamIsCapturing((cudaStream_t)stream, &capture));
  if (capture != cudaStreamCaptureStatusNone) return fail(INFLLM_E_BADARG, "%s: pages change, and the stream captures", what);
  return INFLLM_OK;
}

// the lowest numbers that no sequence has
static int need_seqs(const infllm_pages* p, int64_t n, std::vector<int32_t>* out, const char* what) {
  for (size_t i = 0; i < p->seqs.size() && (int64_t)out->size() < n; ++i)
    if (!p->seqs[i].open) out->push_back((int32_t)i);
  if ((int64_t)out->size() < n)
    return fail(INFLLM_E_CAPACITY, "%s: %lld new sequences, and room for %zu", what, (long long)n, out->size());
  return INFLLM_OK;
}

static void open_seq(infllm_pages* p, int32_t seq) {
  PageSeq& s = p->seqs[seq];
  s.open = true;
  ++s.generation;
  s.length = s.position = 0;
}

// (what sequences share is another thing only where a shared page goes)
static void cut(infllm_pages* p, int32_t seq, int64_t length) {
  PageSeq& s = p->seqs[seq];
  s.changes += s.length != length;
  s.position -= s.length - length;
  s.length = length;
  const size_t left = (size_t)p->pages_of(length);
  while (s.pages.size() > left) {
    p->reshape += p->uses[s.pages.back()] > 1;
    drop_page(p, s.pages.back());
    s.pages.pop_back();
  }
}

// room for counts[i] more tokens of each sequence, or for `same`
static int extend(infllm_pages* p, const int32_t* seqs, const int32_t* counts, int32_t same, int n, void* stream, const char* what) {
  const int page = p->cfg.page_size;
  int64_t need = 0;
  for (int i = 0; i < n; ++i) {
    const PageSeq& s = p->seqs[seqs[i]];
    const int32_t more = counts ? counts[i] : same;
    if (more < 0) return fail(INFLLM_E_BADARG, "%s: %d tokens", what, more);
    if (s.length + more > (int64_t)p->cfg.max_pages * page)
      return fail(INFLLM_E_CAPACITY, "%s: sequence %d would have %lld tokens, and rows of the page table are for %lld", what, seqs[i],
                  (long long)(s.length + more), (long long)p->cfg.max_pages * page);
    if (s.position + more > INT32_MAX) return fail(INFLLM_E_CAPACITY, "%s: positions beyond 31 bits", what);
    need += p->pages_of(s.length + more) - (int64_t)s.pages.size();
    // (as many as would be copied if each of several that share their last page had to: the last one may keep it)
    if (more > 0 && s.length % page && p->uses[s.pages.back()] > 1) ++need;
  }
  INFLLM_TRY(need_pages(p, need, what));
  if (need > 0) INFLLM_TRY(need_stream(p, stream, what));
  ++p->change;
  for (int i = 0; i < n; ++i) {
    PageSeq& s = p->seqs[seqs[i]];
    const int32_t more = counts ? counts[i] : same;
    if (more > 0 && s.length % page && p->uses[s.pages.back()] > 1) {
      const int32_t old = s.pages.back();
      s.pages.back() = take_page(p);
      set_entry(p, seqs[i], s.pages.size() - 1, s.pages.back());
      move_tokens(p, old, 0, s.pages.back(), 0, (int32_t)(s.length % page));
      drop_page(p, old);  // (another one has it still)
      ++p->reshape;
    }
    s.changes += more > 0;
    s.length += more;
    s.position += more;
    const size_t want = (size_t)p->pages_of(s.length);
    while (s.pages.size() < want) {
      s.pages.push_back(take_page(p));
      set_entry(p, seqs[i], s.pages.size() - 1, s.pages.back());
    }
  }
  return INFLLM_OK;
}

int batch_alive(const infllm_page_batch* b, const char* what) {
  if (!b) return fail(INFLLM_E_BADARG, "%s: null pointer", what);
  for (size_t i = 0; i < b->seqs.size(); ++i) {
    const PageSeq& s = b->cache->seqs[b->seqs[i]];
    if (!s.open || s.generation != b->generation[i]) return fail(INFLLM_E_BADARG, "%s: sequence %d of the batch has been freed", what, b->seqs[i]);
  }
  return INFLLM_OK;
}

// Records that a block's last act may be to write: of the process and never given back to the system, since a kernel may outlive its
// cache's books.
namespace {
std::mutex lost_mutex;
std::vector<int32_t*> lost_free;
}  // namespace

static int take_lost(int32_t** out) {
  constexpr int kRecords = 256;
  std::lock_guard<std::mutex> lock(lost_mutex);
  if (lost_free.empty()) {
    lost_free.reserve(kRecords);
    int32_t* block = nullptr;
    INFLLM_CUDA_OK(cudaHostAlloc((void**)&block, kRecords * 4 * sizeof(int32_t), cudaHostAllocPortable));
    for (int i = 0; i < kRecords; ++i) lost_free.push_back(block + 4 * i);
  }
  *out = lost_free.back();
  lost_free.pop_back();
  std::fill(*out, *out + 4, 0);
  return INFLLM_OK;
}

// ------------------------------------------------------------------------------------------------------------ writes
// New tokens' keys and values into their pages, keys and queries rotated to the tokens' positions on the way.  A block has
// a token, or some where a token's rows are few; a thread has 8 dimensions of the first half of a row and the 8 that go with them in the second, so that it needs
// one stretch of the tables for all its rows, and keeps it.  Bound by the bytes of q, k and v, read and written once: 8192 tokens
// of 32 query and 8 KV heads (201 MB) in 40 us, 5.0 TB/s; with blocks of 256 threads 46, of 512 64, with three rows of a thread
// in flight 79 (fewer loads at once for a token of 48 rows).
constexpr int kWriteThreads = 128;
constexpr int kWriteSeqs = 128;  // of a launch

struct WriteParams {
  const char *k, *v, *q;
  char* q_out;                                      // (B, L, n_heads, dim)
  int64_t k_bs, k_hs, k_ts, v_bs, v_hs, v_ts, q_bs, q_hs, q_ts;  // bytes
  char* pages;                                      // of the layer
  const int32_t* table;
  const float *cos_t, *sin_t;                       // null: nothing is rotated
  int64_t plane;                                    // bytes from keys to values
  int32_t max_pages, page, n_kv, n_heads, most, b0, tokens, per_block;  // tokens of the launch, and of a block
  BatchSeq seq[kWriteSeqs];
};

template <typename T>
__device__ __forceinline__ void rotate8(uint4& lo, uint4& hi, const float* cs, const float* sn) {
  T *a = reinterpret_cast<T*>(&lo), *b = reinterpret_cast<T*>(&hi);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // each product rounded to fp32 first, and the sum to 16 bits: as the rotary embedding of the other attention types
    const float x1 = Act<T>::to_f(a[i]), x2 = Act<T>::to_f(b[i]);
    a[i] = Act<T>::from_f(__fadd_rn(__fmul_rn(x1, cs[i]), __fmul_rn(-x2, sn[i])));
    b[i] = Act<T>::from_f(__fadd_rn(__fmul_rn(x2, cs[i]), __fmul_rn(x1, sn[i])));
  }
}

template <typename T, int kDim, bool kRope>
__global__ void __launch_bounds__(kWriteThreads) page_write_kernel(const __grid_constant__ WriteParams P) {
  constexpr int kPer = kDim / 16;  // threads of a row
  const int n_rows = P.n_heads + 2 * P.n_kv, per = min(n_rows * kPer, kWriteThreads);  // threads of a token
  const int sub = (int)threadIdx.x / per, of_token = (int)threadIdx.x - sub * per, token = (int)blockIdx.x * P.per_block + sub;
  if (sub >= P.per_block || token >= P.tokens) return;
  const int b = token / P.most, i = token - b * P.most;
  const BatchSeq S = P.seq[b];
  const int at = i - (P.most - S.count);  // of the new tokens (the shorter sequences' stand at the end)
  const int c = of_token % kPer;
  const int64_t bb = P.b0 + b;
  float cs[8], sn[8];
  if (kRope && at >= 0) {
    const int64_t o = (int64_t)(S.position + at) * (kDim / 2) + c * 8;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      *reinterpret_cast<float4*>(cs + k) = __ldg(reinterpret_cast<const float4*>(P.cos_t + o + k));
      *reinterpret_cast<float4*>(sn + k) = __ldg(reinterpret_cast<const float4*>(P.sin_t + o + k));
    }
  }
  const int place = S.length - S.count + at;
  char* const page_at = at >= 0 ? P.pages + ((int64_t)__ldg(P.table + (int64_t)S.row * P.max_pages + place / P.page) * P.n_kv * P.page + place % P.page) * kDim * 2
                                : nullptr;
  for (int r = of_token / kPer; r < n_rows; r += per / kPer) {
    const char* src;
    char* to;
    const bool is_q = r < P.n_heads, val = r >= P.n_heads + P.n_kv;
    if (is_q) {
      src = P.q + bb * P.q_bs + r * P.q_hs + i * P.q_ts;
      to = P.q_out + ((bb * P.most + i) * P.n_heads + r) * (int64_t)(kDim * 2);
    } else {
      if (at < 0) return;  // (queries come first: nothing is left of this token)
      const int h = r - P.n_heads - (val ? P.n_kv : 0);
      src = val ? P.v + bb * P.v_bs + h * P.v_hs + i * P.v_ts : P.k + bb * P.k_bs + h * P.k_hs + i * P.k_ts;
      to = page_at + (int64_t)h * P.page * kDim * 2 + (val ? P.plane : 0);
    }
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;  // (no token: its query is not one)
    if (at >= 0) {
      lo = *reinterpret_cast<const uint4*>(src + c * 16), hi = *reinterpret_cast<const uint4*>(src + kDim + c * 16);
      if (kRope && !val) rotate8<T>(lo, hi, cs, sn);
    }
    *reinterpret_cast<uint4*>(to + c * 16) = lo;
    *reinterpret_cast<uint4*>(to + kDim + c * 16) = hi;
  }
}

}  // namespace infllm

// ------------------------------------------------------------------------------------------------------- entry points
using namespace infllm;

infllm_pages::~infllm_pages() {
  if (!lost) return;
  std::lock_guard<std::mutex> lock(lost_mutex);
  try {
    lost_free.push_back(lost);
  } catch (const std::bad_alloc&) {  // (16 bytes fewer)
  }
}

extern "C" int infllm_pages_create(const infllm_pages_config* cfg, infllm_pages** out) {
  return guarded("pages_create", [&]() -> int {
    if (!cfg || !out) return fail(INFLLM_E_BADARG, "pages_create: null pointer");
    const infllm_pages_config& c = *cfg;
    if (c.n_layers < 1 || c.n_kv_heads < 1 || c.n_pages < 1 || c.max_sequences < 1 || c.max_pages < 1)
      return fail(INFLLM_E_BADARG, "pages_create: %d layers, %d KV heads, %d pages, %d sequences of %d pages", c.n_layers, c.n_kv_heads,
                  c.n_pages, c.max_sequences, c.max_pages);
    if (c.head_dim != 64 && c.head_dim != 128) return fail(INFLLM_E_UNSUPPORTED, "pages_create: head_dim %d (64 and 128 are built)", c.head_dim);
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
      return fail(INFLLM_E_UNSUPPORTED, "pages_create: pages of %d tokens (16, 32, 64 or 128)", c.page_size);
    if (c.dtype != INFLLM_BF16 && c.dtype != INFLLM_FP16) return fail(INFLLM_E_UNSUPPORTED, "dtype code %d", c.dtype);
    if ((int64_t)c.max_sequences * c.max_pages > INT32_MAX || (int64_t)c.n_layers * 2 * c.n_pages > INT32_MAX ||
        (int64_t)c.n_layers * 2 * c.n_kv_heads * c.page_size * 16 > INT32_MAX || (int64_t)c.max_pages * c.page_size > INT32_MAX)
      return fail(INFLLM_E_BADARG, "pages_create: a page table or a pool beyond 31 bits");
    if (c.device >= 0 && (!c.d_pages || !c.d_table || (uintptr_t)c.d_pages % 16 || (uintptr_t)c.d_table % 4))
      return fail(INFLLM_E_BADARG, "pages_create: the pool has to be 16-byte aligned");
    infllm_pages* p = new infllm_pages();
    p->cfg = c;
    int rc = guarded("pages_create", [&]() -> int {
      p->seqs.resize(c.max_sequences);
      p->uses.resize(c.n_pages, 0);
      p->free_pages.fill(c.n_pages);
      DeviceScope scope(c.device);
      if (!scope.ok()) return fail(INFLLM_E_CUDA, "pages_create: no device %d", c.device);
      if (c.device < 0) return INFLLM_OK;
      INFLLM_CUDA_OK(cudaDeviceGetAttribute(&p->n_sm, cudaDevAttrMultiProcessorCount, c.device));
      INFLLM_TRY(take_lost(&p->lost));
      return pages_encode_map(p);
    });
    if (rc != INFLLM_OK) {
      delete p;
      return rc;
    }
    *out = p;
    return INFLLM_OK;
  });
}

extern "C" int infllm_pages_destroy(infllm_pages* p) {
  delete p;
  return INFLLM_OK;
}

extern "C" int infllm_pages_check(infllm_pages* p, void* stream) {
  return guarded("pages_check", [&]() -> int {
    if (!p) return fail(INFLLM_E_BADARG, "pages_check: null pointer");
    if (!p->lost) return INFLLM_OK;
    DeviceScope scope(p->cfg.device);
    INFLLM_CUDA_OK(cudaStreamSynchronize((cudaStream_t)stream));
    return check_lost(p, (cudaStream_t)stream);
  });
}

extern "C" int infllm_pages_error_set(infllm_pages* p, int code, int where) {
  if (!p || !p->lost) return fail(INFLLM_E_BADARG, "pages_error_set: no cache with a device");
  p->lost[1] = where, p->lost[2] = 0, p->lost[0] = code;
  return INFLLM_OK;
}

extern "C" int infllm_pages_open(infllm_pages* p, int n, int32_t* out) {
  return guarded("pages_open", [&]() -> int {
    if (!p || n < 0 || (n > 0 && !out)) return fail(INFLLM_E_BADARG, "pages_open: null pointer or a negative count");
    std::vector<int32_t> got;
    INFLLM_TRY(need_seqs(p, n, &got, "pages_open"));
    for (int i = 0; i < n; ++i) open_seq(p, out[i] = got[i]);
    return INFLLM_OK;
  });
}

extern "C" int infllm_pages_fork(infllm_pages* p, const int32_t* seqs, int n, int n_each, int32_t* out, void* stream) {
  return guarded("pages_fork", [&]() -> int {
    INFLLM_TRY(check_seqs(p, seqs, n, "pages_fork"));
    if (n_each < 0 || ((int64_t)n * n_each > 0 && !out)) return fail(INFLLM_E_BADARG, "pages_fork: null pointer or a negative count");
    std::vector<int32_t> got;
    INFLLM_TRY(need_seqs(p, (int64_t)n * n_each, &got, "pages_fork"));
    const int page = p->cfg.page_size;
    int64_t need = 0;
    for (int i = 0; i < n; ++i) need += p->seqs[seqs[i]].length % page ? n_each : 0;
    INFLLM_TRY(need_pages(p, need, "pages_fork"));
    DeviceScope scope(p->cfg.device);
    INFLLM_TRY(need_stream(p, stream, "pages_fork"));
    ++p->change;
    int at = 0;
    for (int i = 0; i < n; ++i) {
      const PageSeq& s = p->seqs[seqs[i]];
      const int32_t full = (int32_t)(s.length / page);
      for (int j = 0; j < n_each; ++j, ++at) {
        open_seq(p, got[at]);
        PageSeq& c = p->seqs[got[at]];
        c.length = s.length, c.position = s.position;
        c.pages.assign(s.pages.begin(), s.pages.begin() + full);
        if (full) p->rows.push_back({seqs[i], got[at], full, 0});
        if (s.length % page) {
          c.pages.push_back(take_page(p));
          set_entry(p, got[at], full, c.pages.back());
          move_tokens(p, s.pages[full], 0, c.pages.back(), 0, page);
        }
      }
      for (int32_t k = 0; k < full; ++k) p->uses[s.pages[k]] += n_each;
    }
    std::copy(got.begin(), got.end(), out);
    return flush(p, p, (cudaStream_t)stream);
  });
}

extern "C" int infllm_pages_copy(infllm_pages* p, const int32_t* seqs, int n, infllm_pages* into, int32_t* out, void* stream) {
  return guarded("pages_copy", [&]() -> int {
    INFLLM_TRY(check_seqs(p, seqs, n, "pages_copy"));
    if (!into || (n > 0 && !out)) return fail(INFLLM_E_BADARG, "pages_copy: null pointer");
    const infllm_pages_config &a = p->cfg, &b = into->cfg;
    if (a.n_layers != b.n_layers || a.n_kv_heads != b.n_kv_heads || a.head_dim != b.head_dim || a.page_size != b.page_size || a.dtype != b.dtype || a.device != b.device)
      return fail(INFLLM_E_BADARG, "pages_copy: the caches' pages or devices differ");
    std::vector<int32_t> got;
    INFLLM_TRY(need_seqs(into, n, &got, "pages_copy"));
    int64_t need = 0;
    for (int i = 0; i < n; ++i) {
      const int64_t m = (int64_t)p->seqs[seqs[i]].pages.size();
      if (m > b.max_pages) return fail(INFLLM_E_CAPACITY, "pages_copy: sequence %d has %lld pages, and rows of the page table are for %d", seqs[i], (long long)m, b.max_pages);
      need += m;
    }
    INFLLM_TRY(need_pages(into, need, "pages_copy"));
    DeviceScope scope(b.device);
    INFLLM_TRY(need_stream(into, stream, "pages_copy"));
    ++into->change;
    for (int i = 0; i < n; ++i) {
      const PageSeq& s = p->seqs[seqs[i]];
      open_seq(into, got[i]);
      PageSeq& c = into->seqs[got[i]];
      c.length = s.length, c.position = s.position;
      for (size_t k = 0; k < s.pages.size(); ++k) {
        c.pages.push_back(take_page(into));
        set_entry(into, got[i], k, c.pages.back());
        move_tokens(into, s.pages[k], 0, c.pages.back(), 0, (int32_t)std::min<int64_t>(a.page_size, s.length - (int64_t)k * a.page_size));
      }
    }
    std::copy(got.begin(), got.end(), out);
    return flush(into, p, (cudaStream_t)stream);
  });
}

extern "C" int infllm_pages_truncate(infllm_pages* p, const int32_t* seqs, const int64_t* lengths, int n) {
  return guarded("pages_truncate", [&]() -> int {
    INFLLM_TRY(check_once(p, seqs, n, "pages_truncate"));
    if (n > 0 && !lengths) return fail(INFLLM_E_BADARG, "pages_truncate: null pointer");
    for (int i = 0; i < n; ++i)
      if (lengths[i] < 0 || lengths[i] > p->seqs[seqs[i]].length)
        return fail(INFLLM_E_BADARG, "pages_truncate: %lld of the %lld tokens of sequence %d", (long long)lengths[i],
                    (long long)p->seqs[seqs[i]].length, seqs[i]);
    ++p->change;
    for (int i = 0; i < n; ++i) cut(p, seqs[i], lengths[i]);
    return INFLLM_OK;
  });
}

extern "C" int infllm_pages_free(infllm_pages* p, const int32_t* seqs, int n) {
  return guarded("pages_free", [&]() -> int {
    INFLLM_TRY(check_once(p, seqs, n, "pages_free"));
    ++p->change;
    for (int i = 0; i < n; ++i) {
      cut(p, seqs[i], 0);
      p->seqs[seqs[i]].open = false;
    }
    return INFLLM_OK;
  });
}

extern "C" int infllm_pages_compact(infllm_pages* p, const int32_t* seqs, int n, const int64_t* spans, const int32_t* n_spans, void* stream) {
  return guarded("pages_compact", [&]() -> int {
    INFLLM_TRY(check_once(p, seqs, n, "pages_compact"));
    if (n > 0 && !n_spans) return fail(INFLLM_E_BADARG, "pages_compact: null pointer");
    const int page = p->cfg.page_size, shift = __builtin_ctz(page);
    struct Kept {
      int64_t length;
      int32_t stay;  // pages at the front of which every token stays where it is
    };
    std::vector<Kept> kept(n);
    int64_t need = 0;
    const int64_t* span = spans;
    for (int i = 0; i < n; ++i) {
      if (n_spans[i] < 0 || (n_spans[i] > 0 && !spans)) return fail(INFLLM_E_BADARG, "pages_compact: null pointer or a negative count");
      int64_t at = 0, same = 0, total = 0;
      for (int k = 0; k < n_spans[i]; ++k, span += 2) {
        if (span[0] < at || span[1] < span[0] || span[1] > p->seqs[seqs[i]].length)
          return fail(INFLLM_E_BADARG, "pages_compact: [%lld, %lld) behind %lld, of the %lld tokens of sequence %d", (long long)span[0],
                      (long long)span[1], (long long)at, (long long)p->seqs[seqs[i]].length, seqs[i]);
        if (span[0] == total) same = total + span[1] - span[0];  // (nothing has been left out so far)
        total += span[1] - span[0];
        at = span[1];
      }
      kept[i] = {total, (int32_t)(same / page)};
      need += p->pages_of(total) - kept[i].stay;
    }
    INFLLM_TRY(need_pages(p, need, "pages_compact"));
    DeviceScope scope(p->cfg.device);
    INFLLM_TRY(need_stream(p, stream, "pages_compact"));
    ++p->change, ++p->reshape;
    std::vector<int32_t> gone;
    span = spans;
    for (int i = 0; i < n; ++i) {
      PageSeq& s = p->seqs[seqs[i]];
      const int32_t stay = kept[i].stay;
      std::vector<int32_t> now(s.pages.begin(), s.pages.begin() + stay);
      while ((int64_t)now.size() < p->pages_of(kept[i].length)) {
        now.push_back(take_page(p));
        set_entry(p, seqs[i], now.size() - 1, now.back());
      }
      int32_t to = 0;
      for (int k = 0; k < n_spans[i]; ++k, span += 2) {
        int32_t from = (int32_t)span[0];
        const int32_t stop = (int32_t)span[1];
        // (what stays where it is: up to the end of the pages that are kept)
        if (const int32_t skip = std::min(stop - from, (stay << shift) - to); skip > 0) from += skip, to += skip;
        while (from < stop) {  // up to the end of a page on either side
          const int32_t m = std::min({stop - from, page - (from & (page - 1)), page - (to & (page - 1))});
          move_tokens(p, s.pages[from >> shift], from & (page - 1), now[to >> shift], to & (page - 1), m);
          from += m, to += m;
        }
      }
      gone.insert(gone.end(), s.pages.begin() + stay, s.pages.end());
      s.pages = std::move(now);
      s.changes += s.length != kept[i].length;
      s.length = kept[i].length;
    }
    // (only now: what one sequence leaves must not be taken by the next while it is still to be read)
    for (int32_t g : gone) drop_page(p, g);
    return flush(p, p, (cudaStream_t)stream);
  });
}

extern "C" int infllm_pages_info(const infllm_pages* p, int32_t seq, int64_t* length, int64_t* position) {
  INFLLM_TRY(check_seqs(p, &seq, 1, "pages_info"));
  if (length) *length = p->seqs[seq].length;
  if (position) *position = p->seqs[seq].position;
  return INFLLM_OK;
}

extern "C" int infllm_pages_row(const infllm_pages* p, int32_t seq, int32_t* out, int cap, int* n) {
  INFLLM_TRY(check_seqs(p, &seq, 1, "pages_row"));
  if (!n || cap < 0 || (cap > 0 && !out)) return fail(INFLLM_E_BADARG, "pages_row: null pointer");
  const std::vector<int32_t>& row = p->seqs[seq].pages;
  *n = (int)row.size();
  std::copy(row.begin(), row.begin() + std::min<size_t>(row.size(), (size_t)cap), out);
  return INFLLM_OK;
}

extern "C" int infllm_pages_free_count(const infllm_pages* p) { return p ? p->free_pages.count() : fail(INFLLM_E_BADARG, "pages_free_count: null pointer"); }

extern "C" int infllm_page_batch_create(infllm_pages* p, const int32_t* seqs, int n, infllm_page_batch** out) {
  return guarded("page_batch_create", [&]() -> int {
    if (!out) return fail(INFLLM_E_BADARG, "page_batch_create: null pointer");
    INFLLM_TRY(check_once(p, seqs, n, "page_batch_create"));
    if (n < 1) return fail(INFLLM_E_BADARG, "page_batch_create: no sequences");
    infllm_page_batch* b = new infllm_page_batch();
    int rc = guarded("page_batch_create", [&]() -> int {
      b->cache = p;
      b->seqs.assign(seqs, seqs + n);
      b->count.assign(n, 0);
      for (int i = 0; i < n; ++i) {
        b->generation.push_back(p->seqs[seqs[i]].generation);
        b->as_of.push_back(p->seqs[seqs[i]].changes);
      }
      return INFLLM_OK;
    });
    if (rc != INFLLM_OK) {
      delete b;
      return rc;
    }
    *out = b;
    return INFLLM_OK;
  });
}

extern "C" int infllm_page_batch_destroy(infllm_page_batch* b) {
  delete b;
  return INFLLM_OK;
}

static void set_counts(infllm_page_batch* b, const int32_t* counts, int32_t same) {
  b->most = 0;
  for (size_t i = 0; i < b->seqs.size(); ++i) {
    b->count[i] = counts ? counts[i] : same;
    b->as_of[i] = b->cache->seqs[b->seqs[i]].changes;
    b->most = std::max(b->most, b->count[i]);
  }
  b->plan_of = ~0ull;
}

static void set_reach(const infllm_page_batch* b, int64_t* reach) {
  if (!reach) return;
  *reach = 0;
  for (int32_t s : b->seqs) *reach = std::max(*reach, b->cache->seqs[s].position);
}

extern "C" int infllm_page_batch_extend(infllm_page_batch* b, const int32_t* counts, int32_t same, int64_t* reach, void* stream) {
  return guarded("page_batch_extend", [&]() -> int {
    INFLLM_TRY(batch_alive(b, "page_batch_extend"));
    DeviceScope scope(b->cache->cfg.device);
    INFLLM_TRY(extend(b->cache, b->seqs.data(), counts, same, (int)b->seqs.size(), stream, "page_batch_extend"));
    set_counts(b, counts, same);
    set_reach(b, reach);
    return flush(b->cache, b->cache, (cudaStream_t)stream);
  });
}

// whether every sequence has as many tokens
static int check_counts(const infllm_page_batch* b, const int32_t* counts, int32_t same, const char* what) {
  for (size_t i = 0; i < b->seqs.size(); ++i) {
    const int32_t n = counts ? counts[i] : same;
    const int64_t length = b->cache->seqs[b->seqs[i]].length;
    if (n < 0 || n > length) return fail(INFLLM_E_BADARG, "%s: the newest %d of the %lld tokens of sequence %d", what, n, (long long)length, b->seqs[i]);
  }
  return INFLLM_OK;
}

extern "C" int infllm_page_batch_retract(infllm_page_batch* b, const int32_t* counts, int32_t same) {
  return guarded("page_batch_retract", [&]() -> int {
    INFLLM_TRY(batch_alive(b, "page_batch_retract"));
    INFLLM_TRY(check_counts(b, counts, same, "page_batch_retract"));
    infllm_pages* p = b->cache;
    ++p->change;
    for (size_t i = 0; i < b->seqs.size(); ++i) cut(p, b->seqs[i], p->seqs[b->seqs[i]].length - (counts ? counts[i] : same));
    set_counts(b, nullptr, 0);
    return INFLLM_OK;
  });
}

extern "C" int infllm_page_batch_select(infllm_page_batch* b, const int32_t* counts, int32_t same, int64_t* reach) {
  return guarded("page_batch_select", [&]() -> int {
    INFLLM_TRY(batch_alive(b, "page_batch_select"));
    INFLLM_TRY(check_counts(b, counts, same, "page_batch_select"));
    set_counts(b, counts, same);
    set_reach(b, reach);
    return INFLLM_OK;
  });
}

extern "C" int infllm_page_batch_write(infllm_page_batch* b, int layer, const void* d_k, int64_t k_bs, int64_t k_hs, int64_t k_ts,
                                       const void* d_v, int64_t v_bs, int64_t v_hs, int64_t v_ts, const void* d_q, int64_t q_bs,
                                       int64_t q_hs, int64_t q_ts, void* d_q_out, int n_heads, const float* d_cos, const float* d_sin,
                                       int64_t table_len, void* stream) {
  return guarded("page_batch_write", [&]() -> int {
    INFLLM_TRY(batch_alive(b, "page_batch_write"));
    // (the tokens that the step is about may be gone, and the newest ones others; from here on no sequence is shorter than its count)
    for (size_t i = 0; i < b->seqs.size(); ++i)
      if (b->count[i] > 0 && b->cache->seqs[b->seqs[i]].changes != b->as_of[i])
        return fail(INFLLM_E_BADARG, "page_batch_write: sequence %d has been cut or extended since the step began", b->seqs[i]);
    const infllm_pages_config& c = b->cache->cfg;
    if (c.device < 0) return fail(INFLLM_E_BADARG, "page_batch_write: a cache without a device");
    if (layer < 0 || layer >= c.n_layers) return fail(INFLLM_E_BADARG, "page_batch_write: layer %d of %d", layer, c.n_layers);
    if (b->most > 0 && (!d_k || !d_v || (d_q && (!d_q_out || n_heads < 1)) || (!d_cos) != (!d_sin))) return fail(INFLLM_E_BADARG, "page_batch_write: null pointer");
    if (((uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_q | (uintptr_t)d_q_out | (uintptr_t)d_cos | (uintptr_t)d_sin) % 16 ||
        (k_bs | k_hs | k_ts | v_bs | v_hs | v_ts | q_bs | q_hs | q_ts) % 8)
      return fail(INFLLM_E_BADARG, "page_batch_write: rows must be 16-byte aligned");
    if (b->most == 0) return INFLLM_OK;
    DeviceScope scope(c.device);
    WriteParams P;
    P.k = (const char*)d_k, P.v = (const char*)d_v, P.q = (const char*)d_q;
    P.q_out = (char*)d_q_out;
    P.k_bs = k_bs * 2, P.k_hs = k_hs * 2, P.k_ts = k_ts * 2;
    P.v_bs = v_bs * 2, P.v_hs = v_hs * 2, P.v_ts = v_ts * 2;
    P.q_bs = q_bs * 2, P.q_hs = q_hs * 2, P.q_ts = q_ts * 2;
    P.plane = (int64_t)c.n_pages * c.n_kv_heads * c.page_size * c.head_dim * 2;
    P.pages = (char*)c.d_pages + 2 * layer * P.plane;
    P.table = c.d_table;
    P.cos_t = d_cos, P.sin_t = d_sin;
    P.max_pages = c.max_pages, P.page = c.page_size, P.n_kv = c.n_kv_heads, P.n_heads = d_q ? n_heads : 0, P.most = b->most;
    const int n = (int)b->seqs.size();
    for (int i = 0; i < n; ++i) {
      const PageSeq& s = b->cache->seqs[b->seqs[i]];
      if (d_cos && s.position > table_len) return fail(INFLLM_E_BADARG, "page_batch_write: a rotary table of %lld rows, position %lld", (long long)table_len, (long long)s.position - 1);
      // pages that another sequence has too are not written: a batch that was cut back and selected again is not extended
      if (b->count[i] > 0)
        for (int64_t g = (s.length - b->count[i]) / c.page_size; g < (int64_t)s.pages.size(); ++g)
          if (b->cache->uses[s.pages[g]] > 1) return fail(INFLLM_E_BADARG, "page_batch_write: sequence %d shares the pages of the tokens to be written", b->seqs[i]);
    }
    for (P.b0 = 0; P.b0 < n; P.b0 += kWriteSeqs) {
      const int m = std::min(n - P.b0, kWriteSeqs);
      for (int i = 0; i < m; ++i) {
        const int e = P.b0 + i;
        const PageSeq& s = b->cache->seqs[b->seqs[e]];
        P.seq[i] = {b->seqs[e], (int32_t)s.length, b->count[e], (int32_t)(s.position - b->count[e])};
      }
      if ((int64_t)m * b->most > INT32_MAX) return fail(INFLLM_E_BADARG, "page_batch_write: %lld tokens", (long long)m * b->most);
      P.tokens = m * b->most;
      P.per_block = std::max(1, kWriteThreads / ((P.n_heads + 2 * P.n_kv) * (c.head_dim / 16)));
      const int64_t blocks = ceil_div(P.tokens, P.per_block);
      INFLLM_DISPATCH_DTYPE(c.dtype, T, {
        auto kern = c.head_dim == 128 ? (d_cos ? page_write_kernel<T, 128, true> : page_write_kernel<T, 128, false>)
                                      : (d_cos ? page_write_kernel<T, 64, true> : page_write_kernel<T, 64, false>);
        kern<<<(unsigned)blocks, kWriteThreads, 0, (cudaStream_t)stream>>>(P);
      });
      INFLLM_LAUNCH_OK("page_write_kernel");
    }
    return INFLLM_OK;
  });
}
