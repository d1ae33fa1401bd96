// What the kernels of the attention over a paged cache are given (paged_attn.cu, paged_tc.cu).
#pragma once
#include "pages.cuh"

namespace infllm {

constexpr int kSeeAll = 1 << 30;

struct alignas(16) AttnUnit {
  int32_t row;        // of the page table: one of the node's sequences
  int32_t key0, keys; // keys of the sequence; key0 is the first token of a page
  int32_t lim0;       // a row of token i sees the keys below lim0 + i
  int32_t row0, rows; // of the node's rows: (sequence of the node, token, query head of the KV head)
  int32_t node_seq;   // where the node's sequences are listed
  int32_t hkv;        // KV head, of a unit of many rows; units of few rows are for all of them,
  int32_t part_kv;    // and this many partial rows lie between two heads'
  int32_t part;       // first partial row; -1: the rows are whole, and go to the output
  int32_t pad[2];
};
struct AttnPath {
  int32_t span, tile;  // the node's first row tile, rows of a tile
  int32_t at;          // place of the sequence in the node
};
constexpr int kNearPath = 4;
struct alignas(16) AttnSeq {   // of a sequence of the batch, for the join: its nodes,
  int32_t count, n_path, path; // the first of them here, the others at `path` behind one another
  AttnPath near_path[kNearPath];
  int32_t pad;
};
static_assert(sizeof(AttnSeq) == 64, "");
struct alignas(16) AttnSpan {  // of a row tile of a node and a KV head: n partials of `rows` rows, one behind the other
  int32_t part, n, rows;
  int32_t blocks;     // the rows lie in blocks of 32, four columns of all of them side by side
};

struct PagedParams {
  alignas(64) CUtensorMap map;  // the tensor-core kernel's: all pages as (64 dimensions, token, half of the dimensions, head, page)
  const AttnUnit* tile_unit;
  const int32_t* cta_unit;  // the first unit of each block
  int32_t page0, n_pages;   // the layer's first page in the map, pages from keys to values
  int* err;
  int32_t* lost;            // the cache's own record of it, in the host's memory
  const char* pages;  // keys of the layer
  int64_t plane;      // bytes from keys to values
  const int32_t* table;
  const char* q;
  int64_t q_bs, q_hs, q_ts;  // bytes
  char* out;
  float* lse;
  float *part_o, *part_lse;
  const AttnUnit* unit;
  const AttnSeq* seq;
  const AttnPath* path;
  const AttnSpan* span;
  const int32_t* node_seq;
  int32_t max_pages, page, n_kv, group, most, batch;
  int32_t n_beside;  // units of few rows, by KV heads, for the blocks of many rows
  int32_t after_tiles;
  int32_t* next;     // of those, the next that nobody has taken; the join sets it back
  float scale_log2;
};

// where a row of a node is in the batch
struct RowAt {
  int32_t b, i, h;  // sequence, token, query head of the KV head
};
__device__ __forceinline__ RowAt row_at(const PagedParams& P, int node_seq, int r) {
  RowAt a;
  const int t = r / P.group;
  a.h = r - t * P.group;
  const int j = t / P.most;
  a.i = t - j * P.most;
  a.b = __ldg(P.node_seq + node_seq + j);
  return a;
}

constexpr int kTileRows = 256;  // of a unit of the tensor-core kernel
int paged_tc_launch(const PagedParams& P, int dtype, int head_dim, int n_ctas, cudaStream_t s);

}  // namespace infllm
