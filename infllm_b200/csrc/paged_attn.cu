// Attention of a batch of sequences over a paged cache (pages.cu), with what several of them share read once for all.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij) / sum_j exp(s_ij),  s_ij = scale q_i . k_j,  over the keys j up to query i's place
//
// A batch's pages form a tree: a node is a stretch of pages that the same sequences have.  The queries of all sequences
// under a node, of all query heads of a KV head, are the rows of one product with the node's keys; a query's row appears in
// every node on the way to its sequence, and the parts are joined by their log-sum-exps,
//   M = max_p lse_p,   o = sum_p 2^(lse_p - M) o_p / sum_p 2^(lse_p - M)   (logarithms to base 2).
// A node ends before the newest tokens of its sequences, so that only a sequence's own last stretch (a leaf) has keys that
// some of its queries do not see.
//
// The host knows the tree and all lengths: it cuts every node's rows into tiles and its keys into units of about equal work.
#include <algorithm>
#include <cfloat>
#include <cstring>

#include "attn_tc.cuh"
#include "paged_rows.cuh"

namespace infllm {

using namespace mma;

// A block that gave up a wait has left its rows unwritten: the cache's next call says so, and clears the record.
int check_lost(infllm_pages* p, cudaStream_t s) {
  volatile int32_t* lost = p->lost;
  if (!lost || lost[0] == 0) return INFLLM_OK;
  const int code = lost[0], where = lost[1], block = lost[2];
  lost[0] = 0;
  int* err = nullptr;  // (also where the other kernels have theirs)
  INFLLM_TRY(tc_get_error_ptr(&err));
  INFLLM_CUDA_OK(cudaMemsetAsync(err, 0, 4 * sizeof(int32_t), s));
  return fail(INFLLM_E_TIMEOUT, "a bounded wait of the attention over pages ran out in a call before (code %d, wait %d, block %d): the rows that "
              "the block was to write are not valid", code, where, block);
}

// ------------------------------------------------------------------------------------------------------- few rows
// Four warps share a unit's groups of 16 keys and meet in shared memory.  A token of one sequence over 131072 keys (537 MB, 8 KV heads): 86 us,
// 6.3 TB/s, the join in it.
template <typename T, int kDim, int kNt>
__global__ void __launch_bounds__(kRowWarps * 32, row_blocks(kNt)) paged_rows_kernel(const __grid_constant__ PagedParams P) {
  constexpr int kH = kDim / 64, kPitch = kDim + 4;
  __shared__ __align__(16) float sm_o[kRowWarps][8 * kNt][kPitch];
  __shared__ float sm_m[kRowWarps][8 * kNt], sm_l[kRowWarps][8 * kNt];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const AttnUnit U = P.unit[blockIdx.x];
  const int hkv = blockIdx.y;
  RowsWarp<T, kDim, kNt> W;
  W.find(P, U, hkv);
  // (the kernel before on the stream, where it is the one of many rows, has waited for what was before it by the time this one
  // runs, and leaves other rows: it is waited for at the end, for the join's sake)
  if (P.after_tiles) chain_trigger(); else chain_enter();
  W.begin(P);
  W.template groups<false>(P, U, hkv, warp, kRowWarps);
  W.sums();
  // dimension half*64 + g*8 + i at half*64 + i*8 + g, for the banks' sake
#pragma unroll
  for (int x = 0; x < kNt; ++x) {
    if (t == 0) sm_m[warp][x * 8 + g] = W.m[x], sm_l[warp][x * 8 + g] = W.l[x];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sm_o[warp][x * 8 + 2 * t + e][i * 8 + g] = W.ot[i][x][e];
        if (kH > 1) sm_o[warp][x * 8 + 2 * t + e][64 % kDim + i * 8 + g] = W.ot[i][x][2 + e];
      }
  }
  __syncthreads();
  for (int idx = tid; idx < U.rows * (kDim / 2); idx += kRowWarps * 32) {  // two neighbouring dimensions each
    const int r = idx / (kDim / 2), d = idx % (kDim / 2) * 2;
    const int p0 = (d & 64) | ((d & 7) << 3) | ((d >> 3) & 7), p1 = p0 + 8;
    float mx = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < kRowWarps; ++w) mx = fmaxf(mx, sm_m[w][r]);
    float den = 0.f, n0 = 0.f, n1 = 0.f;
    if (mx != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) {
        const float wt = exp2f(sm_m[w][r] - mx);
        den = fmaf(wt, sm_l[w][r], den);
        n0 = fmaf(wt, sm_o[w][r][p0], n0);
        n1 = fmaf(wt, sm_o[w][r][p1], n1);
      }
      n0 /= den, n1 /= den;
    }
    const float lse = mx == -INFINITY ? -INFINITY : mx + log2f(den);
    if (U.part >= 0) {
      const int64_t pr = (int64_t)U.part + hkv * U.part_kv + r;
      *reinterpret_cast<float2*>(P.part_o + pr * kDim + d) = make_float2(n0, n1);
      if (d == 0) P.part_lse[pr] = lse;
    } else {
      const RowAt a = row_at(P, U.node_seq, U.row0 + r);
      const int64_t orow = ((int64_t)a.b * P.most + a.i) * (P.n_kv * P.group) + hkv * P.group + a.h;
      *reinterpret_cast<uint32_t*>(P.out + (orow * kDim + d) * 2) = pack2<T>(n0, n1);
      if (P.lse && d == 0) P.lse[orow] = lse * (1.f / kLog2e);
    }
  }
  if (P.after_tiles) chain_wait();
}

// ----------------------------------------------------------------------------------------------------------- the join
// kWarps warps per query head and token share the parts of all nodes of its sequence.  Bound by the latency of loads one behind
// the other: where the parts are is looked up before the kernels before on the stream have ended (it is the plan's), and a
// part's row is asked for together with its log-sum-exp, four parts at a time.
template <typename T, int kDim, int kWarps>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ PagedParams P) {
  constexpr int kPer = kDim / 32, kRows = 8 / kWarps, kAhead = 4;
  __shared__ float sm[8][kDim + 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = P.n_kv * P.group;
  const int64_t orow = (int64_t)blockIdx.x * kRows + warp / kWarps;
  const bool in = orow < (int64_t)P.batch * P.most * heads;
  const int h = in ? (int)(orow % heads) : 0, i = in ? (int)(orow / heads % P.most) : 0, b = in ? (int)(orow / heads / P.most) : 0;
  const int hkv = h / P.group;
  const AttnSeq S = P.seq[b];
  const bool is = in && i >= P.most - S.count;  // (a row without a token: zeros)
  auto span_of = [&](const AttnPath& A, int* row) {
    const int r = (A.at * P.most + i) * P.group + h % P.group, tile = r / A.tile;
    *row = r - tile * A.tile;
    return P.span[(A.span + tile) * P.n_kv + hkv];
  };
  int at[kNearPath], n[kNearPath], step[kNearPath];
  bool blocks[kNearPath];
#pragma unroll
  for (int k = 0; k < kNearPath; ++k) {
    at[k] = n[k] = step[k] = 0, blocks[k] = false;
    if (is && k < S.n_path) {
      int r;
      const AttnSpan Z = span_of(S.near_path[k], &r);
      at[k] = Z.part + r, n[k] = Z.n, step[k] = Z.rows, blocks[k] = Z.blocks;
    }
  }
  chain_enter();
  const bool whole = n[0] < 0;  // written by the unit that had all of it
  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
  if (P.n_beside > 0 && blockIdx.x == 0 && threadIdx.x == 0) *P.next = 0;
  auto fold = [&](int first, int count, int stride, bool in_blocks) {  // this warp's of `count` parts
    for (int c0 = warp % kWarps; c0 < count; c0 += kWarps * kAhead) {
      float lse[kAhead], v[kAhead][kPer];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const int c = c0 + e * kWarps;
        lse[e] = -INFINITY;
        if (c >= count) continue;
        const int64_t row = (int64_t)first + (int64_t)c * stride;
        lse[e] = P.part_lse[row];
        const float* o = P.part_o + (in_blocks ? (row & ~(int64_t)31) * kDim + (lane * kPer / 4) * 128 + (row & 31) * 4 + lane * kPer % 4 : row * kDim + lane * kPer);
        if (kPer == 4) *reinterpret_cast<float4*>(v[e]) = *reinterpret_cast<const float4*>(o);
        else *reinterpret_cast<float2*>(v[e]) = *reinterpret_cast<const float2*>(o);
      }
      float mx = m;
#pragma unroll
      for (int e = 0; e < kAhead; ++e) mx = fmaxf(mx, lse[e]);
      const float ref = mx == -INFINITY ? 0.f : mx;  // (a part that is no number is not seen by the maximum)
      const float a = exp2f(m - ref);
      l *= a;
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] *= a;
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        if (lse[e] == -INFINITY) continue;
        const float w = exp2f(lse[e] - ref);
        l += w;
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[k] = fmaf(w, v[e][k], acc[k]);
      }
      m = mx;
    }
  };
#pragma unroll
  for (int k = 0; k < kNearPath; ++k) fold(at[k], n[k], step[k], blocks[k]);
  for (int k = kNearPath; is && k < S.n_path; ++k) {
    int r;
    const AttnSpan Z = span_of(P.path[S.path + k - kNearPath], &r);
    fold(Z.part + r, Z.n, Z.rows, Z.blocks);
  }
  if (kWarps > 1) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) sm[warp][lane * kPer + k] = acc[k];
    if (lane == 0) sm[warp][kDim] = m, sm[warp][kDim + 1] = l;
    __syncthreads();
    if (warp % kWarps) return;
    float mx = m;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sm[warp + w][kDim]);
    const float ms = mx == -INFINITY ? 0.f : mx, a = exp2f(m - ms);
    l *= a;
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] *= a;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float wt = exp2f(sm[warp + w][kDim] - ms);
      l = fmaf(wt, sm[warp + w][kDim + 1], l);
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] = fmaf(wt, sm[warp + w][lane * kPer + k], acc[k]);
    }
    m = mx;
  }
  if (!in || whole) return;
  const float inv = l > 0.f ? 1.f / l : l;  // (a NaN stays one)
  uint32_t* to = reinterpret_cast<uint32_t*>(P.out + (orow * kDim + lane * kPer) * 2);
#pragma unroll
  for (int k = 0; k < kPer; k += 2) to[k / 2] = pack2<T>(acc[k] * inv, acc[k + 1] * inv);
  if (P.lse && lane == 0) P.lse[orow] = l > 0.f ? (m + log2f(l)) * (1.f / kLog2e) : l == 0.f ? -INFINITY : l;
}

template <typename T, int kDim>
static int join_launch(const PagedParams& P, int n_sm, cudaStream_t s) {
  // as many warps to a row as one wave has room for (1024 rows of 23 parts, with the attention: 50.4 us by four warps, 55.4 by eight)
  const int64_t rows = (int64_t)P.batch * P.most * P.n_kv * P.group, warps = n_sm * 32 / std::max<int64_t>(rows, 1);
  auto launch = [&](auto kern, int per_row) { launch_chained(kern, dim3((unsigned)ceil_div(rows * per_row, 8)), dim3(256), 0, s, P); };
  if (warps >= 8) launch(paged_join_kernel<T, kDim, 8>, 8);
  else if (warps >= 4) launch(paged_join_kernel<T, kDim, 4>, 4);
  else if (warps >= 2) launch(paged_join_kernel<T, kDim, 2>, 2);
  else launch(paged_join_kernel<T, kDim, 1>, 1);
  INFLLM_LAUNCH_OK("paged_join_kernel");
  return INFLLM_OK;
}

// ----------------------------------------------------------------------------------------------------------- the plan
namespace {

// Work, in half microseconds
int64_t tile_work(int64_t rows) { return rows > 128 ? 4 : 3; }  // of 128 keys: bound by the products, or by the keys' bytes
constexpr int kUnitWork = 10;  // of a unit of many rows besides its tiles
constexpr int kBlockWork = 8;  // worth a block
constexpr int kGroupWork = 4;  // of a group of 16 keys for few rows, by a warp beside the products

// Work of a batch, in groups of 16 keys by tiles of 16 rows and KV heads, up to which all of it goes to the kernel of few rows: that
// is through before the tensor-core kernel has begun, and is one launch less where both would be needed.  Both ways were timed on 660
// random batches (1 to 64 sequences, prompts of 64 to 60000 tokens, 1 to 64 new ones, six layouts of heads, half with 64 dimensions): the
// time by few rows over that by the tensor cores is, in the median (and from the tenth to the 90th percentile, which says what the measure
// leaves out: keys that several row tiles read, long leaves),
//   work 1500 to 4000    0.70 (0.45 to 0.99)    4000 to 6000    0.81 (0.57 to 1.02)     6000 to 8000    0.88 (0.65 to 1.12)
//        8000 to 10000   1.09 (0.81 to 1.36)    10000 to 13000  1.11 (0.74 to 1.47)     13000 to 20000  1.31 (0.97 to 1.75)
// alike for 64 and 128 dimensions.  With a bound of 7000 a batch takes 3.1 % more than the better way, of 8000 or 8800 2.3 %, of 11000
// 2.5 %, of 14000 3.5 %; always the tensor cores 25 %, never 19 %.
constexpr int64_t kLittle = 8800;

// Groups of 16 keys of a block's unit, where nodes have groups[..] of them for each KV head: so that all blocks run in one, two or
// some waves of as many as the machine holds, whichever is the shortest.  (A sequence of 131072 keys over 32 heads: 449 us by
// 608 blocks where 592 run at once, 319 by 1184.)
int64_t row_chunk(const std::vector<int64_t>& groups, int64_t n_kv, int64_t resident, bool join) {
  // microseconds of a warp's group while all stream, of a block besides, and of the join where only a cut makes one necessary (128
  // sequences of up to 300 keys: 32 us where some are cut, 25 where none is)
  constexpr double kGroup = 3., kBlock = 4., kJoin = 7.;
  int64_t most = kRowWarps, best = kRowWarps;
  for (int64_t g : groups) most = std::max(most, ceil_div(g, kRowWarps) * kRowWarps);
  double least = 1e300;
  auto blocks = [&](int64_t c) {
    int64_t n = 0;
    for (int64_t g : groups) n += std::max<int64_t>(1, ceil_div(g, c * kRowWarps)) * n_kv;
    return n;
  };
  for (int waves = 0; waves <= 6; ++waves) {  // (none: nothing is cut)
    int64_t lo = waves ? 1 : most / kRowWarps, hi = most / kRowWarps;  // the smallest unit with which there are no more blocks than that
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (blocks(mid) <= waves * resident) hi = mid;
      else lo = mid + 1;
    }
    // equal blocks run in waves; where they differ, the short ones fill up what the long ones leave
    double sum = 0.;
    for (int64_t g : groups) {
      const int64_t n = std::max<int64_t>(1, ceil_div(g, lo * kRowWarps));
      sum += (double)(n * n_kv) * ((double)ceil_div(g, n * kRowWarps) * kGroup + kBlock);
    }
    const double longest = lo * kGroup + kBlock;
    const double cost = std::min((double)ceil_div(blocks(lo), resident) * longest, sum / (double)resident + .7 * longest) +
                        (!join && lo * kRowWarps < most ? kJoin : 0.);
    if (cost < least) least = cost, best = lo * kRowWarps;
  }
  return best;
}

struct Node {
  int64_t key0, key1;
  std::vector<int32_t> seqs;  // of the batch
};

// the batch's sequences in the order of their pages, and how many first pages each shares with the one before
void order_batch(infllm_page_batch* b) {
  const infllm_pages* p = b->cache;
  const int n = (int)b->seqs.size();
  auto pages = [&](int i) -> const std::vector<int32_t>& { return p->seqs[b->seqs[i]].pages; };
  b->order.resize(n);
  for (int i = 0; i < n; ++i) b->order[i] = i;
  std::stable_sort(b->order.begin(), b->order.end(), [&](int x, int y) { return pages(x) < pages(y); });
  b->common.assign(n, 0);
  for (int i = 1; i < n; ++i) {
    const std::vector<int32_t>&x = pages(b->order[i - 1]), &y = pages(b->order[i]);
    const size_t most = std::min(x.size(), y.size());
    b->common[i] = (int32_t)(std::mismatch(x.begin(), x.begin() + most, y.begin()).first - x.begin());
  }
}

struct Tree {
  const infllm_page_batch* b;
  std::vector<Node> nodes;
  std::vector<std::vector<int32_t>> path;  // nodes of a sequence of the batch

  int64_t length(int i) const { return b->cache->seqs[b->seqs[i]].length; }
  void add(int64_t key0, int64_t key1, std::vector<int32_t> seqs) {
    for (int32_t i : seqs) path[i].push_back((int32_t)nodes.size());
    nodes.push_back({key0, key1, std::move(seqs)});
  }
  // sequences that share `at` pages; common[k]: pages that seqs[k] shares with seqs[k - 1]
  void build(const std::vector<int32_t>& seqs, const std::vector<int32_t>& common, int32_t at) {
    const int page = b->cache->cfg.page_size;
    size_t k = 0;
    while (k < seqs.size()) {
      // a run of neighbours that have page `at` in common, where it holds none of their newest tokens
      auto whole = [&](size_t x) { return (int32_t)((length(seqs[x]) - b->count[seqs[x]]) / page); };
      std::vector<int32_t> run, with;
      int32_t link = INT32_MAX;
      size_t e = k;
      for (; e < seqs.size(); ++e) {
        if (e > k) link = std::min(link, common[e]);
        if (link <= at) break;
        if (whole(e) > at) {
          run.push_back(seqs[e]);
          with.push_back(run.size() == 1 ? 0 : link);
          link = INT32_MAX;
        } else if (length(seqs[e]) > (int64_t)at * page) {
          add((int64_t)at * page, length(seqs[e]), {seqs[e]});
        }
      }
      k = e;
      if (run.size() == 1) {
        add((int64_t)at * page, length(run[0]), run);
      } else if (run.size() > 1) {
        int32_t to = INT32_MAX;
        for (size_t x = 0; x < run.size(); ++x) {
          to = std::min(to, (int32_t)((length(run[x]) - b->count[run[x]]) / page));
          if (x > 0) to = std::min(to, with[x]);
        }
        add((int64_t)at * page, (int64_t)to * page, run);
        build(run, with, to);
      }
    }
  }
};

template <typename V>
int64_t append(std::vector<int32_t>* plan, const std::vector<V>& v) {
  plan->resize((plan->size() + 3) / 4 * 4);
  const int64_t at = (int64_t)plan->size();
  plan->resize(plan->size() + v.size() * sizeof(V) / 4);
  if (!v.empty()) memcpy(plan->data() + at, v.data(), v.size() * sizeof(V));
  return at;
}

int make_plan(infllm_page_batch* b, int n_heads) {
  const infllm_pages* p = b->cache;
  const int n = (int)b->seqs.size(), n_kv = p->cfg.n_kv_heads, group = n_heads / n_kv, most = b->most;
  if (b->order_of != p->reshape) {
    order_batch(b);
    b->order_of = p->reshape;
  }
  Tree tree{b, {}, std::vector<std::vector<int32_t>>(n)};
  tree.build(b->order, b->common, 0);

  // row tiles: of up to 256 rows for the tensor cores, of up to 16 for nodes that have no more, or where there is little of all
  struct Tile {
    AttnUnit unit;  // of all its keys
    bool many, alone;
  };
  std::vector<Tile> tiles;
  std::vector<int32_t> first_tile, node_seq;
  int64_t few_work = 0, many_work = 0, many_units = 0;  // groups of 16 keys; units of work of the blocks of many rows (tile_work)
  int64_t by_sixteen = 0;
  for (const Node& N : tree.nodes) by_sixteen += ceil_div((int64_t)N.seqs.size() * most * group, kRowTile) * ceil_div(N.key1 - N.key0, 16) * n_kv;
  const bool little = by_sixteen <= kLittle;
  for (const Node& N : tree.nodes) {
    const bool leaf = N.seqs.size() == 1;
    const int64_t rows = (int64_t)N.seqs.size() * most * group;
    const bool many = rows > kRowTile && !little;
    const int size = many ? kTileRows : kRowTile;
    first_tile.push_back((int32_t)tiles.size());
    for (int64_t r = 0; r < rows; r += size) {
      const int32_t in = (int32_t)std::min<int64_t>(size, rows - r);
      // (of a leaf up to the last row's token)
      const int64_t end = leaf ? N.key1 - most + (r + in - 1) / group + 1 : N.key1;
      const int64_t keys = std::max<int64_t>(0, end - N.key0);
      AttnUnit u{b->seqs[N.seqs[0]], (int32_t)N.key0, (int32_t)keys, leaf ? (int32_t)(N.key1 - most + 1) : kSeeAll, (int32_t)r, in, (int32_t)node_seq.size(), 0, 0, -1, {0, 0}};
      tiles.push_back({u, many, leaf && tree.path[N.seqs[0]].size() == 1});
      if (many) many_work += ceil_div(keys, 128) * tile_work(in) * n_kv, many_units += keys > 0 ? n_kv : 0;
      else few_work += ceil_div(keys, 16) * n_kv;
    }
    node_seq.insert(node_seq.end(), N.seqs.begin(), N.seqs.end());
  }

  std::vector<AttnUnit> few, large;
  std::vector<int32_t> cta{0};
  std::vector<AttnSpan> spans(tiles.size() * n_kv);
  int64_t part = 0;
  bool join = false;
  // Few rows.  Two warps of each block of many rows take units of them, whoever is free the next, as much as is done by the time
  // the products are; the rest goes to blocks of four warps, in units of about equal work.
  const int64_t n_cta = many_units ? std::max<int64_t>(1, std::min<int64_t>(p->n_sm, many_work / kBlockWork)) : 0;
  many_work += kUnitWork * (many_units + n_cta);
  int64_t beside_left = n_cta ? 2 * many_work / kGroupWork : 0;
  const int64_t beside_chunk = std::min<int64_t>(16, std::max<int64_t>(2, ceil_div(few_work, 4 * std::max<int64_t>(n_cta, 1)))) * 16;
  std::vector<char> is_beside(tiles.size(), 0);
  std::vector<int64_t> rest;  // groups of the others
  int32_t most_rows = 0;
  bool rest_joins = false;
  for (size_t x = 0; x < tiles.size(); ++x) {
    const Tile& t = tiles[x];
    if (t.many) continue;
    const int64_t groups = ceil_div(t.unit.keys, 16);
    if (groups * n_kv <= beside_left && !(t.alone && groups == 0)) {
      is_beside[x] = 1;
      beside_left -= groups * n_kv;
    } else {
      rest.push_back(groups);
      most_rows = std::max(most_rows, t.unit.rows);
      rest_joins |= !t.alone;
    }
  }
  const int64_t rest_chunk = row_chunk(rest, n_kv, (int64_t)p->n_sm * row_blocks(most_rows > 8 ? 2 : 1), rest_joins || many_units) * 16;
  std::vector<AttnUnit> by_four;
  for (size_t x = 0; x < tiles.size(); ++x) {
    const Tile& t = tiles[x];
    if (t.many) continue;
    const int64_t keys = t.unit.keys;
    const bool beside = is_beside[x];
    const int64_t chunk = beside ? beside_chunk : rest_chunk, cut = ceil_div(keys, chunk), each = cut ? ceil_div(ceil_div(keys, 16), cut) * 16 : 0;
    std::vector<AttnUnit>& to = beside ? few : by_four;
    AttnUnit u = t.unit;
    if (!beside && t.alone && cut <= 1) {
      to.push_back(u);
      for (int h = 0; h < n_kv; ++h) spans[x * n_kv + h].n = -1;
      continue;
    }
    u.part_kv = (int32_t)(cut * u.rows);
    for (int h = 0; h < n_kv; ++h) spans[x * n_kv + h] = {(int32_t)(part + h * cut * u.rows), (int32_t)cut, u.rows, 0};
    for (int64_t k = 0; k < keys; k += each) {
      u.key0 = t.unit.key0 + (int32_t)k, u.keys = (int32_t)std::min(each, keys - k), u.part = (int32_t)(part + k / each * u.rows);
      to.push_back(u);
    }
    part += cut * u.rows * n_kv;
    join = true;
  }
  const size_t n_beside = few.size();
  few.insert(few.end(), by_four.begin(), by_four.end());
  // many rows: one list of all key tiles, cut into as many stretches of equal work as there are SMs, or fewer
  int64_t done = 0;  // work that has been dealt out
  for (size_t x = 0; x < tiles.size(); ++x) {
    const Tile& t = tiles[x];
    if (!t.many) continue;
    const int64_t n_tiles = ceil_div(t.unit.keys, 128), weight = tile_work(t.unit.rows);
    for (int h = 0; h < n_kv; ++h) {
      AttnUnit u = t.unit;
      u.hkv = h;
      const size_t first = large.size();
      for (int64_t k = 0; k < n_tiles || (k == 0 && t.alone);) {
        // up to the end of the block's share; what is left of one tile or less goes along, and the last block takes all that is left
        const bool last = (int64_t)cta.size() >= n_cta;
        const int64_t share = last ? many_work : ceil_div(many_work * (int64_t)cta.size(), n_cta);
        int64_t take = std::min(n_tiles - k, std::max<int64_t>(0, (share - done - kUnitWork) / weight));
        if (last || n_tiles - k - take <= 1) take = n_tiles - k;
        if (take > 0 || n_tiles == 0) {
          u.key0 = t.unit.key0 + (int32_t)k * 128;
          u.keys = (int32_t)std::min<int64_t>(take * 128, t.unit.keys - k * 128);
          large.push_back(u);
        }
        k += take, done += take > 0 ? take * weight + kUnitWork : 0;
        if (n_tiles == 0) break;
        if (!last && (k < n_tiles || done >= share)) cta.push_back((int32_t)large.size());
      }
      const size_t cut = large.size() - first;
      AttnSpan& z = spans[x * n_kv + h];
      if (cut == 1 && t.alone) {
        z.n = -1;
        continue;
      }
      const int32_t room = (u.rows + 31) / 32 * 32;
      part = (part + 31) / 32 * 32;
      z = {(int32_t)part, (int32_t)cut, room, 1};
      for (size_t k = first; k < large.size(); ++k, part += room) large[k].part = (int32_t)part;
      join = true;
    }
  }
  if (part > INT32_MAX) return fail(INFLLM_E_BADARG, "page_batch_plan: too many partial rows");
  b->n_ctas = large.empty() ? 0 : (int32_t)cta.size();
  cta.push_back((int32_t)large.size());
  std::vector<AttnSeq> seqs;
  std::vector<AttnPath> paths;
  for (int i = 0; i < n; ++i) {
    AttnSeq q{};
    q.count = b->count[i], q.path = (int32_t)paths.size();
    join |= tree.path[i].empty();
    for (int32_t x : tree.path[i]) {
      const Node& N = tree.nodes[x];
      const int32_t tile = (int64_t)N.seqs.size() * most * group > kRowTile && !little ? kTileRows : kRowTile;
      const AttnPath a{first_tile[x], tile, (int32_t)(std::find(N.seqs.begin(), N.seqs.end(), i) - N.seqs.begin())};
      if (q.n_path < kNearPath) q.near_path[q.n_path] = a;
      else paths.push_back(a);
      ++q.n_path;
    }
    seqs.push_back(q);
  }
  b->plan.assign(4, 0);  // the number of the next unit of few rows, and nothing
  b->off_unit = append(&b->plan, few);
  b->off_tile_unit = append(&b->plan, large);
  b->off_cta = append(&b->plan, cta);
  b->off_seq = append(&b->plan, seqs);
  b->off_path = append(&b->plan, paths);
  b->off_span = append(&b->plan, spans);
  b->off_node_seq = append(&b->plan, node_seq);
  b->n_row_units = (int32_t)by_four.size();
  b->n_beside = (int32_t)n_beside;
  b->most_rows = most_rows;
  b->join = join;
  b->part_rows = part;
  return INFLLM_OK;
}

}  // namespace

}  // namespace infllm

using namespace infllm;

static int64_t plan_room(const infllm_page_batch* b) { return ((int64_t)b->plan.size() * 4 + 255) / 256 * 256; }

extern "C" int infllm_page_batch_plan(infllm_page_batch* b, int n_heads, int64_t* work_bytes) {
  return guarded("page_batch_plan", [&]() -> int {
    INFLLM_TRY(batch_alive(b, "page_batch_plan"));
    const infllm_pages* p = b->cache;
    if (!work_bytes) return fail(INFLLM_E_BADARG, "page_batch_plan: null pointer");
    if (n_heads < 1 || n_heads % p->cfg.n_kv_heads) return fail(INFLLM_E_BADARG, "page_batch_plan: %d query heads over %d KV heads", n_heads, p->cfg.n_kv_heads);
    if ((int64_t)b->most * n_heads * (int64_t)b->seqs.size() > INT32_MAX) return fail(INFLLM_E_BADARG, "page_batch_plan: more than 2^31 query rows");
    for (size_t i = 0; i < b->seqs.size(); ++i)
      if (b->count[i] > p->seqs[b->seqs[i]].length)
        return fail(INFLLM_E_BADARG, "page_batch_plan: the newest %d tokens of sequence %d, which has %lld", b->count[i], b->seqs[i],
                    (long long)p->seqs[b->seqs[i]].length);
    b->plan_of = ~0ull;
    INFLLM_TRY(make_plan(b, n_heads));
    b->plan_of = p->change;
    b->plan_heads = n_heads;
    b->upload = true;
    *work_bytes = plan_room(b) + b->part_rows * (p->cfg.head_dim + 4) * 4;
    return INFLLM_OK;
  });
}

extern "C" int infllm_page_batch_attend(infllm_page_batch* b, int layer, const void* d_q, int64_t q_bs, int64_t q_hs, int64_t q_ts, void* d_out,
                                        float* d_lse, int n_heads, float scale, void* d_work, void* stream) {
  return guarded("page_batch_attend", [&]() -> int {
    INFLLM_TRY(batch_alive(b, "page_batch_attend"));
    infllm_pages* p = b->cache;
    const infllm_pages_config& c = p->cfg;
    if (c.device < 0) return fail(INFLLM_E_BADARG, "page_batch_attend: a cache without a device");
    if (layer < 0 || layer >= c.n_layers) return fail(INFLLM_E_BADARG, "page_batch_attend: layer %d of %d", layer, c.n_layers);
    // (maxima are taken of the scores before they are scaled)
    if (!(scale >= 0.f) || !(scale * kLog2e <= FLT_MAX)) return fail(INFLLM_E_BADARG, "page_batch_attend: a scale of %g", (double)scale);
    if (b->plan_of != p->change || b->plan_heads != n_heads) return INFLLM_PAGES_NO_PLAN;
    if (b->most == 0) return INFLLM_OK;
    if (!d_q || !d_out || !d_work) return fail(INFLLM_E_BADARG, "page_batch_attend: null pointer");
    if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_work) % 16 || (q_bs | q_hs | q_ts) % 8)
      return fail(INFLLM_E_BADARG, "page_batch_attend: rows must be 16-byte aligned");
    // (a row's place in the queries is counted in 16 bytes, in 31 bits)
    const int64_t far = std::max<int64_t>((int64_t)b->seqs.size() - 1, 0) * q_bs + (int64_t)(n_heads - 1) * q_hs + (int64_t)(b->most - 1) * q_ts;
    if (q_bs < 0 || q_hs < 0 || q_ts < 0 || far / 8 > INT32_MAX) return fail(INFLLM_E_BADARG, "page_batch_attend: queries that lie %lld bytes apart", (long long)far * 2);
    DeviceScope scope(c.device);
    cudaStream_t s = (cudaStream_t)stream;
    INFLLM_TRY(check_lost(p, s));
    if (b->upload) {
      // (a copy that is captured is not made, and would be made later of whatever the next plan leaves there)
      cudaStreamCaptureStatus capture;
      INFLLM_CUDA_OK(cudaStreamIsCapturing(s, &capture));
      if (capture != cudaStreamCaptureStatusNone) return fail(INFLLM_E_BADARG, "page_batch_attend: a plan that is not on the device yet, on a stream that captures");
      INFLLM_CUDA_OK(cudaMemcpyAsync(d_work, b->plan.data(), b->plan.size() * 4, cudaMemcpyHostToDevice, s));
    }
    b->upload = false;
    PagedParams P;
    P.plane = (int64_t)c.n_pages * c.n_kv_heads * c.page_size * c.head_dim * 2;
    P.pages = (const char*)c.d_pages + 2 * layer * P.plane;
    P.table = c.d_table;
    P.q = (const char*)d_q, P.q_bs = q_bs * 2, P.q_hs = q_hs * 2, P.q_ts = q_ts * 2;
    P.out = (char*)d_out, P.lse = d_lse;
    P.part_o = (float*)((char*)d_work + plan_room(b)), P.part_lse = P.part_o + b->part_rows * c.head_dim;
    const int32_t* plan = (const int32_t*)d_work;
    P.unit = (const AttnUnit*)(plan + b->off_unit), P.seq = (const AttnSeq*)(plan + b->off_seq);
    P.path = (const AttnPath*)(plan + b->off_path), P.span = (const AttnSpan*)(plan + b->off_span), P.node_seq = plan + b->off_node_seq;
    P.map = p->map;
    P.tile_unit = (const AttnUnit*)(plan + b->off_tile_unit), P.cta_unit = plan + b->off_cta;
    P.page0 = 2 * layer * c.n_pages, P.n_pages = c.n_pages;
    INFLLM_TRY(tc_get_error_ptr(&P.err));
    P.lost = p->lost;
    P.max_pages = c.max_pages, P.page = c.page_size, P.n_kv = c.n_kv_heads, P.group = n_heads / c.n_kv_heads, P.most = b->most;
    P.batch = (int)b->seqs.size();
    P.n_beside = b->n_beside * c.n_kv_heads;
    P.next = (int32_t*)d_work;
    // (the tensor-core kernel masks scores before they are scaled: -inf times 0 is no number.  By the least normal number instead, scores
    // of less than 2^100 are zeros beside any reference)
    P.scale_log2 = std::max(scale * kLog2e, FLT_MIN);
    if (b->n_ctas > 0) INFLLM_TRY(paged_tc_launch(P, c.dtype, c.head_dim, b->n_ctas, s));
    INFLLM_DISPATCH_DTYPE(c.dtype, T, {
      if (b->n_row_units > 0) {
        P.unit += b->n_beside, P.after_tiles = b->n_ctas > 0;
        auto kern = c.head_dim == 128 ? (b->most_rows <= 8 ? paged_rows_kernel<T, 128, 1> : paged_rows_kernel<T, 128, 2>)
                                      : (b->most_rows <= 8 ? paged_rows_kernel<T, 64, 1> : paged_rows_kernel<T, 64, 2>);
        launch_chained(kern, dim3(b->n_row_units, c.n_kv_heads), dim3(kRowWarps * 32), 0, s, P);
        INFLLM_LAUNCH_OK("paged_rows_kernel");
      }
      if (b->join) INFLLM_TRY((c.head_dim == 128 ? join_launch<T, 128>(P, p->n_sm, s) : join_launch<T, 64>(P, p->n_sm, s)));
    });
    return INFLLM_OK;
  });
}
