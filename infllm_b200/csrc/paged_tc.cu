// Attention over shared pages for many rows (paged_attn.cu has the formulas): tcgen05 products, S and O in TMEM, keys and values by TMA.
//
// A unit is up to 256 rows of one KV head (two tiles of 128: one each for two teams of four softmax warps, a thread per row)
// by a stretch of keys.  Both teams' products read the same key tile, which halves the bytes from L2; while one team works out
// its exponentials the tensor pipe forms the other's products.  S of a team and its P, which takes S's place in TMEM and is
// the A operand of P V from there, have 128 columns, O another 128.  A unit of up to 128 rows has one team, whose S goes to the
// two buffers in turn, so that the next product runs while it works; such units are bound by the bytes of the keys.
// A warp asks for pages, one box of a page and operand (boxes of 16 to 64 tokens: one per lane), through a ring of tiles in
// the order K0 K1 V0 K2 V1 ..; another warp issues the products.  Blocks work through a list of units of about equal work.
// Two more warps take units of few rows (paged_rows.cuh), whose loads fit in beside the products.
// The reference maximum of a row is lazy: it moves when the maximum has grown by 2^8, and only then O is scaled.
// P is one 16-bit number: the A operand is 16 bits, and a second one for what is left over would be half as many products again.  With
// the output's own rounding that is an error of 2.3e-3 for bf16 where that alone is 1.7e-3.  Sums, O and partial rows are fp32.
//
// What bounds it: with two teams a round of one of them, 3450 cycles for 256 rows by 128 keys (by clock readings, 2048 tokens behind 28000:
// maximum 300, exponentials 1490, hand-overs 270, then its P V and next Q K^T, 512 each, and 360 until the scores are seen), in which the
// tensor pipe is needed for 2048; with one team the keys' bytes.  128 tokens of 32/8 heads over 131072 shared keys: 283 us for 275 GFLOP
// as a launch by itself (0.97 PFLOP/s; each byte from HBM once, though two blocks share every key), 337 with the join, calls back to
// back; 32 over 32768 (134 MB): 40 us, of which 8 lie before the first scores and 3 between the last tile and its rows.
// Tried: steps of 64 keys with two buffers of scores a team (a product of 64 columns takes nearly as long as one of 128: 13 % more time), P in
// two halves (scores 350 cycles earlier, exponentials 700 longer), an issuer that polls both teams (25 % more), sixteen softmax warps (5 to
// 18 % more).
#include <atomic>
#include <type_traits>

#include "paged_rows.cuh"
#include "attn_tc.cuh"
#include "ring.cuh"
#include "tc_softmax.cuh"

namespace infllm {

namespace ptc {
constexpr int kStages = 5;
constexpr int kThreads = 12 * 32;
constexpr int kWarpTma = 8, kWarpMma = 9, kWarpRows = 10;  // the last two: units of few rows
enum { FULL0 = 0, EMPTY0 = FULL0 + kStages, Q_FULL0 = EMPTY0 + kStages, S_FULL0 = Q_FULL0 + 2, P_FULL0 = S_FULL0 + 3, PV_DONE0 = P_FULL0 + 3, N_BARS = PV_DONE0 + 3 };
// Scores and what follows from them go by channels: 0 and 1 are the teams' with the buffer of the same number, 2 is the first
// team's with the second buffer.  (The second team may be a unit ahead, one that it has no part in: on a barrier that both
// teams use in turn it would take the other's phase for its own.)
__device__ __forceinline__ int channel(bool two, int team, int i) { return two ? team : (i & 1) * 2; }
__device__ __forceinline__ int buffer(int channel) { return channel ? 1 : 0; }
template <int kDim>
struct Smem {
  static constexpr int kTileBytes = 128 * kDim * 2;  // of 128 rows, as one or two swizzled tiles of 64 dimensions
  static constexpr int kQ = 0, kRing = 2 * kTileBytes, kBar = kRing + kStages * kTileBytes, kTotal = kBar + 256;
};
// position of a key tile and of a value tile of a unit of n tiles in the ring
__device__ __forceinline__ int pos_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int pos_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }
}  // namespace ptc

template <typename T, int kDim>
__global__ void __launch_bounds__(ptc::kThreads, 1) paged_tc_kernel(const __grid_constant__ PagedParams P) {
  using namespace ptc;
  using L = Smem<kDim>;
  constexpr int kHalves = kDim / 64;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t s_base = smem_u32(smem), sQ = s_base + L::kQ, sRing = s_base + L::kRing, bars = s_base + L::kBar;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBar + N_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBar + N_BARS * 8 + 8);
  auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    static_assert(N_BARS <= 32 && N_BARS * 8 + 16 <= 256, "");
    if (lane < N_BARS) mbar_init(bar(lane), lane == Q_FULL0 || lane == Q_FULL0 + 1 || (lane >= P_FULL0 && lane < P_FULL0 + 3) ? 4u : 1u);
    if (lane == 0) *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kWarpTma && lane == 0) tma_prefetch_map(&P.map);
  if (warp == kWarpMma) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  constexpr uint32_t idesc_qk = make_idesc(kBf16, 128, 128, false), idesc_pv = make_idesc(kBf16, 128, kDim, true);
  const int u0 = P.cta_unit[blockIdx.x], u1 = P.cta_unit[blockIdx.x + 1];

  // (the plan is there: the roles wait for the kernels before on the stream where they first need what those have written)
  if (warp == kWarpTma) {
    // ======================================================================================================== pages
    chain_enter();
    const bool lead = elect_one();
    const int per = 128 / P.page;  // pages of a tile
    int slot = 0;
    bool ok = true;
    for (int u = u0; u < u1 && ok; ++u) {
      const AttnUnit U = P.tile_unit[u];
      const int n = (U.keys + 127) / 128, first = U.key0 / P.page, n_pages = (U.keys + P.page - 1) / P.page;
      const int32_t* row = P.table + (int64_t)U.row * P.max_pages + first;
      auto ids = [&](int i) { return lane < per && i * per + lane < n_pages ? __ldg(row + i * per + lane) : 0; };
      auto load = [&](int i, int id, int plane) {
        const int b = slot % kStages;
        if (slot >= kStages) ok = warp_wait(bar(EMPTY0 + b), ring_parity(slot - kStages, kStages), abort_flag, P.err, 701);
        if (!ok) return;
        const int there = min(per, n_pages - i * per);
        const uint32_t to = sRing + b * L::kTileBytes;
        if (lead) mbar_expect_tx(bar(FULL0 + b), there * P.page * kDim * 2);
        __syncwarp();
        const int at = P.page0 + plane * P.n_pages;
        if (per == 1) {  // both halves of the dimensions in one box
          if (lead) tma_load_5d(to, &P.map, bar(FULL0 + b), 0, 0, 0, U.hkv, at + id);
        } else {
          const int pg = lane / kHalves, h = lane % kHalves, mine = __shfl_sync(0xffffffffu, id, pg);
          if (pg < there) tma_load_5d(to + h * kSubTileBytes + pg * P.page * 128, &P.map, bar(FULL0 + b), 0, 0, h, U.hkv, at + mine);
        }
        __syncwarp();
        ++slot;
      };
      int now = ids(0), next = ids(1);
      if (per == 1) now = __shfl_sync(0xffffffffu, now, 0);
      for (int i = 0; i < n && ok; ++i) {
        // K one tile ahead of V
        if (i == 0) load(0, now, 0);
        int after = 0;
        if (per == 1) next = __shfl_sync(0xffffffffu, next, 0);
        if (ok && i + 1 < n) {
          after = ids(i + 2);
          load(i + 1, next, 0);
        }
        if (ok) load(i, now, 1);
        now = next, next = after;
      }
    }
    // nothing is on its way to this block, nor will be signalled in it, when it goes: the releases come behind all products
    for (int b = 0; b < kStages && ok; ++b) {
      const int last = ring_last(slot, kStages, b);
      if (last >= 0) ok = warp_wait(bar(EMPTY0 + b), ring_parity(last, kStages), abort_flag, P.err, 702);
    }
    if (!ok && lane == 0) {  // given up: loads on their way get a bounded chance to land
      for (int b = 0; b < kStages; ++b) {
        const int last = ring_last(slot, kStages, b);
        for (uint32_t w = 0; last >= 0 && w < 4096 && !mbar_try_wait(bar(FULL0 + b), ring_parity(last, kStages)); ++w) __nanosleep(64);
      }
    }
    __syncwarp();
  } else if (warp == kWarpMma) {
    // ===================================================================================================== products
    const bool lead = elect_one();
    int base = 0, np[3] = {0, 0, 0}, n_one = 0, n_two = 0;  // ring position, probabilities that have been waited for, units of each team
    bool ok = true;
    const uint64_t ring_k = make_sdesc(sRing, 16, 1024), ring_v = make_sdesc(sRing, kSubTileBytes, 1024), qd0 = make_sdesc(sQ, 16, 1024);
    auto arrived = [&](int pos) { ok = ok && warp_wait(bar(FULL0 + pos % kStages), ring_parity(pos, kStages), abort_flag, P.err, 711); };
    auto release = [&](int pos) {
      if (lead) tc_commit(bar(EMPTY0 + pos % kStages));
    };
    auto qk = [&](int q, int pos, int ch) {  // S of a team's queries
      if (lead) {
        const uint64_t qd = qd0 + (uint64_t)(q * L::kTileBytes >> 4), kd = ring_k + (uint64_t)((pos % kStages) * L::kTileBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks) {
          const uint64_t o = (uint64_t)(((ks >> 2) * kSubTileBytes + (ks & 3) * 32) >> 4);
          mma_ss(tmem + buffer(ch) * 128, qd + o, kd + o, idesc_qk, ks > 0);
        }
        tc_commit(bar(S_FULL0 + ch));
      }
      __syncwarp();
    };
    auto pv = [&](int team, int pos, int ch, bool first) {
      ok = ok && warp_wait(bar(P_FULL0 + ch), np[ch] & 1, abort_flag, P.err, 712);
      ++np[ch];
      if (!ok) return;
      tc_fence_after();
      if (lead) {
        const uint64_t vd = ring_v + (uint64_t)((pos % kStages) * L::kTileBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) mma_ts(tmem + 256 + team * 128, tmem + buffer(ch) * 128 + 8 * ks, vd + (uint64_t)((ks * 2048) >> 4), idesc_pv, !first || ks > 0);
        tc_commit(bar(PV_DONE0 + ch));
      }
      __syncwarp();
    };
    for (int u = u0; u < u1 && ok; ++u) {
      const AttnUnit U = P.tile_unit[u];
      const int n = (U.keys + 127) / 128, tail = U.keys - (n - 1) * 128;
      const bool two = U.rows > 128;
      if (n == 0) continue;  // (rows that see no key; nothing holds the softmax warps back from the next unit's queries)
      ok = warp_wait(bar(Q_FULL0), n_one++ & 1, abort_flag, P.err, 710);
      if (two) ok = ok && warp_wait(bar(Q_FULL0 + 1), n_two++ & 1, abort_flag, P.err, 710);
      if (!ok) break;
      auto values = [&](int i) {
        const int pos = base + pos_v(i, n);
        arrived(pos);
        if (ok && i == n - 1 && tail < 128) {
          // behind the last key may be anything, NaN too, and the product has 0 times it: zeros instead
          for (int h = 0; h < kHalves; ++h)
            for (int o = tail * 128 + lane * 16; o < kSubTileBytes; o += 32 * 16)
              *reinterpret_cast<uint4*>(smem + L::kRing + (pos % kStages) * L::kTileBytes + h * kSubTileBytes + o) = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        return pos;
      };
      const int ahead = two ? 1 : 2;  // a team's buffers
      for (int i = 0; i < ahead && i < n && ok; ++i) {
        const int pos = base + pos_k(i);
        arrived(pos);
        if (!ok) break;
        tc_fence_after();
        qk(0, pos, channel(two, 0, i));
        if (two) qk(1, pos, 1);
        release(pos);
      }
      for (int i = 0; i < n && ok; ++i) {
        const int pv_pos = values(i), more = i + ahead, k_pos = base + pos_k(more);
        if (!ok) break;
        if (two) {
          pv(0, pv_pos, 0, i == 0);
          if (ok && more < n) {
            arrived(k_pos);
            if (ok) qk(0, k_pos, 0);
          }
          if (ok) pv(1, pv_pos, 1, i == 0);
          if (!ok) break;
          release(pv_pos);
          if (more < n) {
            qk(1, k_pos, 1);
            release(k_pos);
          }
        } else {
          pv(0, pv_pos, channel(false, 0, i), i == 0);
          if (!ok) break;
          release(pv_pos);
          if (more < n) {
            arrived(k_pos);
            if (!ok) break;
            qk(0, k_pos, channel(false, 0, more));
            release(k_pos);
          }
        }
      }
      base += 2 * n;
    }
    __syncwarp();
  } else if (warp >= kWarpRows) {
    // ===================================================================================================== few rows
    chain_wait();
    // (whoever is free takes the next: the products beside them keep some waiting longer)
    while (true) {
      int j = P.n_beside;
      if (lane == 0 && j > 0) j = atomicAdd(P.next, 1);
      j = __shfl_sync(0xffffffffu, j, 0);
      if (j >= P.n_beside) break;
      const AttnUnit U = P.unit[j / P.n_kv];
      if (U.rows <= 8) {
        RowsWarp<T, kDim, 1> W;
        W.alone(P, U, j % P.n_kv);
      } else {
        RowsWarp<T, kDim, 2> W;
        W.alone(P, U, j % P.n_kv);
      }
    }
    __syncwarp();
  } else {
    // ====================================================================================================== softmax
    const int quad = warp & 3, team = warp >> 2, row = quad * 32 + lane;
    const uint32_t lane_base = ((uint32_t)(quad * 32)) << 16;
    const uint32_t tO = tmem + 256 + team * 128 + lane_base;
    struct Turn {  // a unit of this team's, and this thread's row of it
      int u, n, key0, rows, lim, all;
      bool two, whole;
      int64_t out;  // row of the output, or of the partial results
      int q;  // 16-byte pieces from the first query's first row to its own, -1: none
    };
    auto find = [&](int u) {  // the team's next unit from u on: of the plan alone
      Turn t{u, 0, 0, 0, 0, 0, false, false, 0, -1};
      for (; t.u < u1; ++t.u)
        if (team == 0 || __ldg(&P.tile_unit[t.u].rows) > 128) break;
      if (t.u >= u1) return t;
      const AttnUnit U = P.tile_unit[t.u];
      t.n = (U.keys + 127) / 128, t.key0 = U.key0, t.two = U.rows > 128, t.whole = U.part < 0;
      t.rows = min(128, U.rows - team * 128);
      t.lim = U.key0 + U.keys;  // rows that are none are not masked, so that whole tiles stay whole: nothing of them is written
      if (row < t.rows) {
        const RowAt at = row_at(P, U.node_seq, U.row0 + team * 128 + row);
        t.lim = at.i < P.most - __ldg(&P.seq[at.b].count) ? 0 : min(t.lim, U.lim0 + at.i);
        t.q = (int)((at.b * P.q_bs + (int64_t)(U.hkv * P.group + at.h) * P.q_hs + at.i * P.q_ts) / 16);
        t.out = t.whole ? ((int64_t)at.b * P.most + at.i) * (P.n_kv * P.group) + U.hkv * P.group + at.h : (int64_t)U.part + team * 128 + row;
      }
      t.all = __reduce_min_sync(0xffffffffu, t.lim);
      return t;
    };
    auto queries = [&](const Turn& t) {
      // The warp's 32 rows, 16 bytes a lane, swizzled as TMA would have them.  No product reads the last unit's any more: its
      // scores have been seen.  (Rolled, and past the registers: a unit waits for the instructions of what runs once, and
      // for one load; unrolled over 16 registers this took 5 us instead of 1.5.)
      constexpr int kPer = kDim / 8, kAt = 32 / kPer;
      const int c = lane % kPer;
      const uint32_t to = sQ + team * L::kTileBytes + quad * 32 * 128 + (c >> 3) * kSubTileBytes;
#pragma unroll 1
      for (int r = lane / kPer; r < 32; r += kAt) {
        const int from = __shfl_sync(0xffffffffu, t.q, r);
        mma::cp_async16(to + r * 128 + (((c & 7) ^ (r & 7)) << 4), P.q + (int64_t)max(from, 0) * 16 + c * 16, from >= 0);
      }
      mma::cp_async_commit();
      mma::cp_async_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Q_FULL0 + team));
    };
    int ns[3] = {0, 0, 0};  // tiles so far of each channel
    bool ok = true;
    Turn now = find(u0);
    chain_wait();
    if (now.n > 0) queries(now);
    while (now.u < u1 && ok) {
      const Turn next = find(now.u + 1);
      const int step = now.two ? 1 : 2;
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < now.n && ok; ++i) {
        const int ch = channel(now.two, team, i);
        const uint32_t tS = tmem + buffer(ch) * 128 + lane_base;
        ok = warp_wait(bar(S_FULL0 + ch), (ns[ch] + i / step) & 1, abort_flag, P.err, 720);
        if (!ok) break;
        tc_fence_after();
        const int j0 = now.key0 + i * 128;
        if (now.all < j0 + 128) {
          // what a row does not see is taken out of the scores where they are
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            const int hi = now.lim - j0 - c;
            if (__all_sync(0xffffffffu, hi >= 32)) continue;
            uint32_t w[32];
            tmem_ld32(tS + c, w);
            tmem_wait_ld32(w);
#pragma unroll
            for (int k = 0; k < 32; ++k) w[k] = k < hi ? w[k] : 0xff800000u;
            tmem_st32(tS + c, w);
          }
          tmem_wait_st();
        }
        float s[32], mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        uint32_t* us = reinterpret_cast<uint32_t*>(s);
        {
          float b[32];
          uint32_t* ub = reinterpret_cast<uint32_t*>(b);
          tmem_ld32(tS + 32, ub);
          tmem_ld32(tS + 64, us);
          tmem_wait_ld32(ub);
          tmem_wait_ld32(us);
          max_chunk(b, mx);
          tmem_ld32(tS + 96, ub);
          max_chunk(s, mx);
          tmem_ld32(tS, us);
          tmem_wait_ld32(ub);
          tmem_wait_ld32(us);
          max_chunk(b, mx);
          max_chunk(s, mx);
        }
        const float mt = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]) * P.scale_log2;
        const float mn = mt - m > 8.f ? mt : m;  // (from -inf: any number)
        const float alpha = m == -INFINITY ? 1.f : ex2_approx(m - mn);
        const bool scale_o = __any_sync(0xffffffffu, mn != m && m != -INFINITY) && i > 0;
        l *= alpha;
        m = mn;
        const float nm = m == -INFINITY ? 0.f : -m;
        float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // P, packed, takes the place of scores that have been read: 16 columns for 32
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float2 e[16];
          uint32_t pk[16];
          arg_chunk(s, P.scale_log2, nm, e);
          tmem_ld32_if(c < 3, tS + 32 * c + 32, us);
          exp_chunk<T, 5>(e, rs, pk);
          tmem_st16(tS + 16 * c, pk);
          tmem_wait_ld32(us);
        }
        const float2 r = fadd2(fadd2(rs[0], rs[1]), fadd2(rs[2], rs[3]));
        const float sum = r.x + r.y;
        l += m == -INFINITY && sum < 1.f ? 0.f : sum;  // (the polynomial leaves 2^-126 of a masked key; a NaN stays one)
        if (scale_o) {
          // O has the products up to the tile before: wait for the last of them
          const int pb = channel(now.two, team, i - 1);
          ok = warp_wait(bar(PV_DONE0 + pb), (ns[pb] + (i - 1) / step) & 1, abort_flag, P.err, 721);
          if (!ok) break;
          tc_fence_after();
          const float2 al = make_float2(alpha, alpha);
#pragma unroll 1
          for (int c = 0; c < kDim; c += 32) {
            uint32_t o[32];
            tmem_ld32(tO + c, o);
            tmem_wait_ld32(o);
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float2 x = fmul2(make_float2(__uint_as_float(o[k]), __uint_as_float(o[k + 1])), al);
              o[k] = __float_as_uint(x.x), o[k + 1] = __float_as_uint(x.y);
            }
            tmem_st32(tO + c, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL0 + ch));
      }
      // the next unit's queries first, so that its first scores are formed while this one's rows are written
      if (ok && next.n > 0) queries(next);
      if (ok && now.n > 0) {
        const int pb = channel(now.two, team, now.n - 1);
        ok = warp_wait(bar(PV_DONE0 + pb), (ns[pb] + (now.n - 1) / step) & 1, abort_flag, P.err, 722);
      }
      if (ok) {
        tc_fence_after();
        const float inv = l > 0.f ? 1.f / l : l;  // (a NaN stays one)
#pragma unroll 1
        for (int c = 0; c < kDim; c += 32) {
          uint32_t o[32];
          float* f = reinterpret_cast<float*>(o);
          if (now.n > 0) {
            tmem_ld32(tO + c, o);
            tmem_wait_ld32(o);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0;
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) f[k] *= inv;
          if (row < now.rows && !now.whole) {
            // partial rows lie in blocks of 32, four columns of all of them side by side: every store is one stretch
            float4* to = reinterpret_cast<float4*>(P.part_o + (now.out - lane) * kDim) + (c / 4) * 32 + lane;
#pragma unroll
            for (int k = 0; k < 8; ++k) to[k * 32] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
          } else if (row < now.rows) {
            uint4* to = reinterpret_cast<uint4*>(P.out + (now.out * kDim + c) * 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                typename Act<T>::T2 v = Act<T>::from_f2(f[8 * k + 2 * e], f[8 * k + 2 * e + 1]);
                w[e] = *reinterpret_cast<uint32_t*>(&v);
              }
              to[k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          __syncwarp();
        }
        if (row < now.rows) {
          const float lse = l > 0.f ? m + log2f(l) : l == 0.f ? -INFINITY : l;
          if (!now.whole) P.part_lse[now.out] = lse;
          else if (P.lse) P.lse[now.out] = lse * (1.f / kLog2e);
        }
        tc_fence_before();
      }
      if (now.two) ns[team] += now.n;
      else ns[0] += (now.n + 1) / 2, ns[2] += now.n / 2;
      __syncwarp();
      now = next;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) {
    volatile int32_t* lost = P.lost;
    lost[1] = *(volatile int*)(P.err + 1), lost[2] = blockIdx.x;
    __threadfence_system();
    lost[0] = kErrWaitTimeout;
  }
}

int paged_tc_launch(const PagedParams& P, int dtype, int head_dim, int n_ctas, cudaStream_t s) {
  INFLLM_DISPATCH_DTYPE(dtype, T, {
    auto kern = head_dim == 128 ? paged_tc_kernel<T, 128> : paged_tc_kernel<T, 64>;
    const int smem = (head_dim == 128 ? ptc::Smem<128>::kTotal : ptc::Smem<64>::kTotal) + 1024;
    static std::atomic<uint64_t> set[2];  // devices that know it, per head_dim (and, by the dispatch, type)
    int dev = 0;
    INFLLM_CUDA_OK(cudaGetDevice(&dev));
    std::atomic<uint64_t>& there = set[head_dim == 128];
    if (dev >= 64 || !(there.load(std::memory_order_relaxed) >> dev & 1)) {
      INFLLM_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      if (dev < 64) there.fetch_or(1ull << dev);
    }
    launch_chained(kern, dim3(n_ctas), dim3(ptc::kThreads), smem, s, P);
  });
  INFLLM_LAUNCH_OK("paged_tc_kernel");
  return INFLLM_OK;
}

// all pages of all layers, keys and values, as (64 dimensions, token, half of the dimensions, head, page)
int pages_encode_map(infllm_pages* p) {
  const infllm_pages_config& c = p->cfg;
  const uint64_t halves = c.head_dim / 64, row = (uint64_t)c.head_dim * 2;
  const uint64_t dims[5] = {64, (uint64_t)c.page_size, halves, (uint64_t)c.n_kv_heads, (uint64_t)c.n_layers * 2 * c.n_pages};
  const uint64_t strides[4] = {row, 128, row * c.page_size, row * c.page_size * c.n_kv_heads};
  const uint32_t box[5] = {64, (uint32_t)c.page_size, c.page_size == 128 ? (uint32_t)halves : 1u, 1, 1};
  return encode_tensor_map(&p->map, c.dtype, c.d_pages, 5, dims, strides, box);
}

}  // namespace infllm
