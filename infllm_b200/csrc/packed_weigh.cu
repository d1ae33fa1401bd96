// The weights of the tokens of the cache in 4 bits, for many rows (packed_attn.cu has the formulas): sums of the columns of the attention
// probabilities, whose log-sum-exps are known, w_j = sum_i exp2(s_ij - lse_i).
//
// S^T = K Q^T by tcgen05: keys are the lanes of TMEM, so that a thread has a key and adds up along its row, and nothing is exchanged.  A
// unit is 256 keys of one KV head (two tiles of 128, one each for two teams of eight warps, of which four have half of the columns each)
// by the counted rows that see them, 128 at a time: keys are taken out of their codes once, queries go through a ring of tiles with their
// log-sum-exps.  Units are dealt out to the blocks in stretches of about equal work, as (unit, tile of rows); what is cut is added up by
// one more kernel, in order.
// Sums: within a tile of rows in eight numbers of 32 bits, then tile by tile, so that an error does not grow with the rows.
// What bounds it: what is issued around the exponentials, 32768 of them in 3000 cycles (a prompt of 4096 tokens, 32/8 heads: 115 us; with a
// quarter of them by a quintic on the FMA pipe instead of an eighth 118, three eighths 125; without any 80).  By clock readings a warp is
// at its sums for 2330 cycles of a tile, the loads' copies take 1700, the products' issue 1100.  Tried: keys as the operand in TMEM, a warp of
// its own for each team's products, products of 64 columns (each as long); eight warps of sums instead of sixteen (5 % more).
#include <atomic>

#include "attn_tc.cuh"
#include "packed_attn.cuh"
#include "ring.cuh"
#include "tc_softmax.cuh"

namespace infllm {

namespace xwg {
constexpr int kStages = 4;
constexpr int kSumWarps = 16, kWarpMma = 16, kWarpLoad = 17, kLoadWarps = 4;  // eight warps of a team: four for each half of the columns
constexpr int kThreads = (kWarpLoad + kLoadWarps) * 32;
enum { FULL0 = 0, EMPTY0 = FULL0 + kStages, K_FULL = EMPTY0 + kStages, K_FREE, S_FULL0, S_FREE0 = S_FULL0 + 4, SUMS = S_FREE0 + 4, SUMS_READ, N_BARS };  // S: 2 * team + buffer
template <int kDim>
struct Smem {
  static constexpr int kTileBytes = 128 * kDim * 2;
  static constexpr int kK = 0, kRing = 2 * kTileBytes, kLse = kRing + kStages * kTileBytes, kBar = kLse + kStages * 512, kSum = kBar + 256, kTotal = kSum + kWeighKeys * 4;
};

struct Piece {
  int b, hkv, key0, keys;  // up to 256 keys
  int row0, n;             // rows row0 + 128 * i ..
  int slot;                // of partial sums, -1: the unit is whole
};
struct Pieces {  // a block's, in turn
  int u, t, ue, te, slot;
  __device__ __forceinline__ explicit Pieces(const PackedTcParams& P) {
    const int2 a = P.start[blockIdx.x], z = P.start[blockIdx.x + 1];
    u = a.x, t = a.y, ue = z.x, te = z.y, slot = 2 * blockIdx.x;
  }
  __device__ __forceinline__ bool next(const PackedTcParams& P, Piece& p) {
    if (u > ue || (u == ue && t >= te)) return false;
    p.b = seq_of(P.a, u);
    const PackedAttnSeq& S = P.a.seq[p.b];
    const int local = u - S.unit0, block = local % S.chunks;
    p.hkv = local / S.chunks;
    p.key0 = block * kWeighKeys, p.keys = min(kWeighKeys, S.length - p.key0);
    const int all = weigh_tiles(S, P.a.group, P.a.weigh, block), end = u == ue ? te : all;
    p.row0 = weigh_row0(S, P.a.group, P.a.weigh, block) + t * 128, p.n = end - t;
    p.slot = t == 0 && end == all ? -1 : slot;
    slot = 2 * blockIdx.x + 1;
    if (end == all) ++u, t = 0;
    else t = end;
    return true;
  }
};

// exponentials to base 2 of eight pairs, added up: one pair on the FMA pipe
__device__ __forceinline__ void exp_sum(const float2* a, float2* rs) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 p = k == 7 ? ex2_poly2<5>(a[k]) : make_float2(ex2_approx(a[k].x), ex2_approx(a[k].y));
    rs[k & 3] = fadd2(rs[k & 3], p);
  }
}
}  // namespace xwg

__device__ __forceinline__ void tmem_ld16_if(bool yes, uint32_t taddr, uint32_t* r) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %17, 0;\n\t"
      "@p tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t}"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
      : "r"(taddr), "r"((uint32_t)yes)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               ::"memory");
}

template <typename T, int kDim>
__global__ void __launch_bounds__(xwg::kThreads, 1) packed_weigh_tc_kernel(const __grid_constant__ PackedTcParams P) {
  using namespace xwg;
  using L = Smem<kDim>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t s_base = smem_u32(smem), sK = s_base + L::kK, sRing = s_base + L::kRing, bars = s_base + L::kBar;
  float* const sLse = reinterpret_cast<float*>(smem + L::kLse);  // log-sum-exps of a tile's rows, negative
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBar + N_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBar + N_BARS * 8 + 8);
  auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* const err = P.a.err;

  if (warp == 0) {
    static_assert(N_BARS <= 32 && N_BARS * 8 + 16 <= 256, "");
    // tiles and keys: the four warps that load; free tiles: the products and the warps that sum; free scores: a team's; sums: half of them
    if (lane < N_BARS) mbar_init(bar(lane), lane < EMPTY0 || lane == K_FULL ? 4u : lane < K_FULL ? kSumWarps + 1u : lane >= S_FREE0 ? kSumWarps / 2u : 1u);
    if (lane == 0) *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr uint32_t idesc = make_idesc(kBf16, 128, 128, false);
  chain_enter();
  Pieces pieces(P);
  Piece U;
  bool ok = true;

  if (warp >= kWarpLoad) {
    // ================================================================================================ keys and queries
    using C = Codes<T>;
    constexpr int kGroups = kDim / 32, kStep = 128 / kGroups;
    const int at = (warp - kWarpLoad) * 32 + lane, t = at % kGroups, r0 = at / kGroups;
    int slot = 0, n_pieces = 0;
    while (ok && pieces.next(P, U)) {
      const PackedAttnSeq& S = P.a.seq[U.b];
      if (n_pieces > 0) ok = warp_wait(bar(K_FREE), (n_pieces - 1) & 1, abort_flag, err, 781);
      if (!ok) break;
      ++n_pieces;
      const int64_t row = P.a.at.row0(S.slot, U.hkv) + U.key0;
      const char* codes = P.a.at.codes + row * (kDim / 2);
      const char* scales = P.a.at.scales + row * (kDim / 8);
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        uint4 c[kGroups];
        uint32_t ms[kGroups];
#pragma unroll
        for (int x = 0; x < kGroups; ++x) {
          const int k = tile * 128 + r0 + x * kStep;
          c[x] = make_uint4(0, 0, 0, 0), ms[x] = 0;
          if (k < U.keys) {
            c[x] = __ldg(reinterpret_cast<const uint4*>(codes + k * (kDim / 2) + t * 16));
            ms[x] = __ldg(reinterpret_cast<const uint32_t*>(scales + k * (kDim / 8) + t * 4));
          }
        }
        unsigned char* to = smem + L::kK + tile * L::kTileBytes + (t >> 1) * kSubTileBytes;
#pragma unroll
        for (int x = 0; x < kGroups; ++x) put_group<T>(to, r0 + x * kStep, t, c[x], ms[x]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(K_FULL));

      // query tiles, one on its way behind the one that has to be there
      const int rows = S.count * P.a.group;
      const int64_t q0 = (int64_t)(P.a.b0 + U.b) * P.a.q_bs + (int64_t)U.hkv * P.a.group * P.a.q_hs + (int64_t)(P.a.most - S.count) * P.a.q_ts;
      const float* row_lse = P.a.row_lse + ((int64_t)(P.a.b0 + U.b) * P.a.at.n_kv + U.hkv) * P.a.most * P.a.group;
      constexpr int kPer = kDim / 8, kAt = 32 / kPer, kLag = 1;
      const int c = lane % kPer, wq = (warp - kWarpLoad) * 32;
      const int step_h = kAt % P.a.group;
      const int64_t step = (int64_t)(kAt / P.a.group) * P.a.q_ts + step_h * P.a.q_hs, wrap = P.a.q_ts - P.a.group * P.a.q_hs;
      // (a row's log-sum-exp is asked for a tile ahead: a tile is not to wait for it)
      auto lse_of = [&](int r) { return r < rows ? -__ldg(row_lse + r) : -INFINITY; };  // (a row that is none gives nothing)
      float z = lse_of(U.row0 + wq + lane);
      for (int i = 0; i < U.n + kLag && ok; ++i) {
        if (i < U.n) {
          const float next = lse_of(U.row0 + (i + 1) * 128 + wq + lane);
          const int b = (slot + i) % kStages;
          if (slot + i >= kStages) ok = warp_wait(bar(EMPTY0 + b), ring_parity(slot + i - kStages, kStages), abort_flag, err, 782);
          if (!ok) break;
          sLse[b * 128 + wq + lane] = z;
          z = next;
          // a lane's rows are kAt apart: the next one is some heads on, and a token where those are through
          const uint32_t to = sRing + b * L::kTileBytes + wq * 128 + (c >> 3) * kSubTileBytes;
          const int r = U.row0 + i * 128 + wq + lane / kPer, tok = r / P.a.group, left = rows - r;
          int h = r - tok * P.a.group;
          const char* from = P.a.q + q0 + (int64_t)h * P.a.q_hs + (int64_t)tok * P.a.q_ts + c * 16;
#pragma unroll
          for (int x = 0; x < 32; x += kAt) {
            const int row = x + lane / kPer;
            mma::cp_async16(to + row * 128 + (((c & 7) ^ (row & 7)) << 4), x < left ? from : P.a.q, x < left);
            from += step, h += step_h;
            if (h >= P.a.group) h -= P.a.group, from += wrap;
          }
        }
        mma::cp_async_commit();  // (an empty one behind the last)
        if (i >= kLag) {
          mma::cp_async_wait<kLag>();
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(FULL0 + (slot + i - kLag) % kStages));
        }
      }
      slot += U.n;
    }
    mma::cp_async_wait<0>();
    // nothing will be signalled in this block when it goes
    for (int b = 0; b < kStages && ok; ++b) {
      const int last = ring_last(slot, kStages, b);
      if (last >= 0) ok = warp_wait(bar(EMPTY0 + b), ring_parity(last, kStages), abort_flag, err, 783);
    }
    if (ok && n_pieces > 0) ok = warp_wait(bar(K_FREE), (n_pieces - 1) & 1, abort_flag, err, 784);
    __syncwarp();
  } else if (warp == kWarpMma) {
    // ===================================================================================================== products
    const bool lead = elect_one();
    const uint64_t kd0 = make_sdesc(sK, 16, 1024), qd0 = make_sdesc(sRing, 16, 1024);
    int slot = 0, n_pieces = 0, used[4] = {0, 0, 0, 0};
    while (ok && pieces.next(P, U)) {
      ok = warp_wait(bar(K_FULL), n_pieces++ & 1, abort_flag, err, 791);
      const int teams = U.keys > 128 ? 2 : 1;
      for (int i = 0; i < U.n && ok; ++i, ++slot) {
        ok = warp_wait(bar(FULL0 + slot % kStages), ring_parity(slot, kStages), abort_flag, err, 792);
        for (int team = 0; team < teams && ok; ++team) {
          const int s = 2 * team + (slot & 1);
          if (used[s] > 0) ok = warp_wait(bar(S_FREE0 + s), (used[s] - 1) & 1, abort_flag, err, 793);
          if (!ok) break;
          ++used[s];
          tc_fence_after();
          if (lead) {
#pragma unroll
            for (int ks = 0; ks < kDim / 16; ++ks) {
              const uint64_t o = (uint64_t)(((ks >> 2) * kSubTileBytes + (ks & 3) * 32) >> 4);
              mma_ss(tmem + s * 128, kd0 + (uint64_t)(team * L::kTileBytes >> 4) + o, qd0 + (uint64_t)((slot % kStages) * L::kTileBytes >> 4) + o, idesc, ks > 0);
            }
            tc_commit(bar(S_FULL0 + s));
          }
          __syncwarp();
        }
        if (ok && lead) tc_commit(bar(EMPTY0 + slot % kStages));
        __syncwarp();
      }
      if (ok && lead) tc_commit(bar(K_FREE));
      __syncwarp();
    }
  } else {
    // ========================================================================================================= sums
    const int quad = warp & 3, team = warp >> 2 & 1, half = warp >> 3;  // (a warp's place among four says which lanes of TMEM it reads)
    const uint32_t lane_base = ((uint32_t)(quad * 32)) << 16;
    int slot = 0, used[2] = {0, 0}, n_units = 0;
    while (ok && pieces.next(P, U)) {
      const PackedAttnSeq& S = P.a.seq[U.b];
      const bool mine = team == 0 || U.keys > 128;
      const int k = team * 128 + quad * 32 + lane, j = U.key0 + k;
      const int first = max(0, j - (S.length - S.count)) * P.a.group;  // row that sees this thread's key
      const int last_first = __reduce_max_sync(0xffffffffu, k < U.keys ? first : 0);
      float sum = 0.f;
      for (int i = 0; i < U.n && ok; ++i, ++slot) {
        const int stage = slot % kStages, buf = slot & 1, s = 2 * team + buf;
        ok = warp_wait(bar(FULL0 + stage), ring_parity(slot, kStages), abort_flag, err, 795);  // (for the log-sum-exps)
        if (ok && mine) {
          ok = warp_wait(bar(S_FULL0 + s), used[buf]++ & 1, abort_flag, err, 796);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tS = tmem + s * 128 + lane_base + half * 64;
          const int row0 = U.row0 + i * 128 + half * 64;
          const float4* lse = reinterpret_cast<const float4*>(sLse + stage * 128 + half * 64);
          float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 sc = make_float2(P.a.scale_log2, P.a.scale_log2);
          uint32_t w[16];
          tmem_ld16_if(true, tS, w);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            tmem_wait_ld16(w);
            float2 a[8];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float4 z = lse[c * 4 + x];
              a[2 * x] = ffma2(__uint_as_float(w[4 * x]), __uint_as_float(w[4 * x + 1]), sc, make_float2(z.x, z.y));
              a[2 * x + 1] = ffma2(__uint_as_float(w[4 * x + 2]), __uint_as_float(w[4 * x + 3]), sc, make_float2(z.z, z.w));
            }
            tmem_ld16_if(c < 3, tS + 16 * c + 16, w);
            if (last_first > row0 + 16 * c) {
              const int hidden = first - row0 - 16 * c;  // columns of rows that do not see the key
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                if (2 * x < hidden) a[x].x = -INFINITY;
                if (2 * x + 1 < hidden) a[x].y = -INFINITY;
              }
            }
            exp_sum(a, rs);
          }
          tmem_wait_ld();
          tc_fence_before();
          const float2 r = fadd2(fadd2(rs[0], rs[1]), fadd2(rs[2], rs[3]));
          sum += r.x + r.y;
        }
        __syncwarp();
        if (lane == 0) {
          if (mine) mbar_arrive(bar(S_FREE0 + s));
          mbar_arrive(bar(EMPTY0 + stage));
        }
      }
      // the second half's sums go to the first half's warps
      float* const halves = reinterpret_cast<float*>(smem + L::kSum);
      if (half == 1) {
        if (ok && n_units > 0) ok = warp_wait(bar(SUMS_READ), (n_units - 1) & 1, abort_flag, err, 797);
        if (ok) halves[k] = sum;
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(bar(SUMS));
      } else {
        ok = ok && warp_wait(bar(SUMS), n_units & 1, abort_flag, err, 798);
        if (ok) sum += halves[k];
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(bar(SUMS_READ));
      }
      ++n_units;
      if (ok && half == 0 && k < U.keys) {
        if (U.slot >= 0) {
          P.a.part_o[(int64_t)U.slot * kWeighKeys + k] = sum;
        } else {
          float* to = P.a.weights + P.a.at.row0(S.slot, U.hkv) + j;
          *to = P.a.decay == 0.f ? sum : P.a.decay * *to + sum;
        }
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) tmem_dealloc(tmem, 512);
}

// what units that were cut have given, in order
__global__ void __launch_bounds__(kWeighKeys) packed_weigh_join_kernel(const __grid_constant__ PackedTcParams P) {
  const int b = blockIdx.z, hkv = blockIdx.y, block = blockIdx.x, key = block * kWeighKeys + threadIdx.x;
  const PackedAttnSeq S = P.a.seq[b];
  chain_enter();
  if (S.count == 0 || key >= S.length) return;
  const int unit = S.unit0 + hkv * S.chunks + block, first = block_of(P, unit, 0);
  const int parts = block_of(P, unit, weigh_tiles(S, P.a.group, P.a.weigh, block) - 1) - first + 1;
  if (parts == 1) return;
  float sum = 0.f;
  for (int c = 0; c < parts; ++c) sum += P.a.part_o[(int64_t)(2 * (first + c) + (P.start[first + c].x < unit)) * kWeighKeys + threadIdx.x];
  float* to = P.a.weights + P.a.at.row0(S.slot, hkv) + key;
  *to = P.a.decay == 0.f ? sum : P.a.decay * *to + sum;
}

int packed_weigh_tc_launch(const PackedTcParams& P, int dtype, int head_dim, bool join, int longest, cudaStream_t s) {
  INFLLM_DISPATCH_DTYPE(dtype, T, {
    auto kern = head_dim == 128 ? packed_weigh_tc_kernel<T, 128> : packed_weigh_tc_kernel<T, 64>;
    const int smem = (head_dim == 128 ? xwg::Smem<128>::kTotal : xwg::Smem<64>::kTotal) + 1024;
    static std::atomic<uint64_t> set[2];  // devices that know it, per head_dim (and, by the dispatch, type)
    int dev = 0;
    INFLLM_CUDA_OK(cudaGetDevice(&dev));
    std::atomic<uint64_t>& there = set[head_dim == 128];
    if (dev >= 64 || !(there.load(std::memory_order_relaxed) >> dev & 1)) {
      INFLLM_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (dev < 64) there.fetch_or(1ull << dev);
    }
    INFLLM_CUDA_OK(launch_chained(kern, dim3(P.n_ctas), dim3(xwg::kThreads), smem, s, P));
  });
  INFLLM_LAUNCH_OK("packed_weigh_tc_kernel");
  if (join) {
    INFLLM_CUDA_OK(launch_chained(packed_weigh_join_kernel, dim3((unsigned)ceil_div(longest, kWeighKeys), P.a.at.n_kv, P.a.batch), dim3(kWeighKeys), 0, s, P));
    INFLLM_LAUNCH_OK("packed_weigh_join_kernel");
  }
  return INFLLM_OK;
}

}  // namespace infllm
