// Attention over the cache in 4 bits for many rows (packed_attn.cu has the formulas): tcgen05 products of numbers that six warps
// take out of their codes, S and O in TMEM.
//
// A unit is up to 256 rows of one KV head by a stretch of keys.  Two teams of four softmax warps, a thread per row, have 128 rows each;
// of up to 128 rows both have all, and take the key tiles in turn: each with a maximum, a sum and an O of its own, which are put
// together at the unit's end, where a thread reads the other team's O of its row from TMEM.  (A tile is in a team's hands for 1.1 us:
// with one team that, not its bytes, would be a tile's time.)
// Six more warps bring codes from global memory through registers, and leave 16-bit numbers, swizzled as the products want them, in a
// ring of tiles in the order K0 K1 V0 K2 V1 ..; both teams' products read the same tile, so that it is taken out once for 256 rows.
// (Eight of them, with softmax in pieces of 16 columns to do with 96 registers: of 48 rows 4 % less, of 192 rows 8 % more.)  Prompts'
// tiles, which many blocks of rows read, are taken out once for all of them by a kernel before, and fetched by one warp.
// Another warp issues the products.  S of a team and its P, which takes S's place in TMEM and is the A operand of P V from there, have 128
// columns, O another 128.  The reference of a row is lazy (packed_attn.cuh): only where it moves O is scaled.
// P is one 16-bit number: the A operand is 16 bits, and a second one for what is left over would be half as many products again.  (bf16: off by
// up to 2^-8 of itself.  fp16: by 2^-11 of itself, and where it is less than 2^-25 of its row's largest, by up to 2^-36 of that.)
// Sums, O and partial rows are fp32.
// What bounds it: the softmax warps' chain (scores out of TMEM, maximum, exponentials, P back) between two products of its team, with six code
// warps beside it for issue.  2048 tokens behind 28000, 32/8 heads of 128 in bf16: 889 us with the image, 2.2 us for a tile of 256 rows by
// 128 keys (products alone, with P as it lies there, 1.63; as fast as they can be issued, 1.1 to 1.2), 963 without.  48 tokens of 8
// sequences of 12288 (192 rows of 8 KV heads) 124 us, 12 tokens (48 rows) 77.
// Tried: 4, 7, 8, 10, 12, 14 and 16 code warps; registers given from warpgroup to warpgroup with 28 warps (five times slower: spills).
#include <atomic>
#include <climits>

#include "attn_tc.cuh"
#include "decode_warp.cuh"
#include "packed_attn.cuh"
#include "ring.cuh"
#include "tc_softmax.cuh"

namespace infllm {

namespace xtc {
constexpr int kStages = 5;
// Warps: eight of softmax; six that take numbers out of their codes (half of them keys, half values), or one that fetches tiles that are
// there already (kImage); one that issues products.  Sixteen or fewer, so that a thread has 128 registers.
constexpr int kWarpCodes = 8, kCodeWarps = 6;
constexpr int makers(bool image) { return image ? 1 : kCodeWarps; }
constexpr int threads(bool image) { return (kWarpCodes + makers(image) + 1) * 32; }
enum { FULL0 = 0, EMPTY0 = FULL0 + kStages, Q_FULL0 = EMPTY0 + kStages, S_FULL0 = Q_FULL0 + 2, P_FULL0 = S_FULL0 + 2, PV_DONE0 = P_FULL0 + 2, MERGE = PV_DONE0 + 2, N_BARS };
template <int kDim>
struct Smem {
  static constexpr int kTileBytes = 128 * kDim * 2;  // of 128 rows, as one or two swizzled tiles of 64 dimensions
  static constexpr int kQ = 0, kRing = 2 * kTileBytes, kBar = kRing + kStages * kTileBytes, kMl = kBar + 256, kTotal = kMl + 2 * 128 * 8;
};
// position of a key tile and of a value tile of a unit of n tiles in the ring, and what is at a position
__device__ __forceinline__ int pos_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int pos_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }
__device__ __forceinline__ bool is_value(int p, int n) { return p == 2 * n - 1 || (p > 0 && p % 2 == 0); }
__device__ __forceinline__ int tile_at(int p, int n) { return p == 2 * n - 1 ? n - 1 : p % 2 ? (p + 1) / 2 : p == 0 ? 0 : p / 2 - 1; }

struct Piece {  // of a unit: what a block has of it
  int b, hkv, row0, rows;  // rows of the sequence's new tokens, up to 256
  int tile0, n, keys;      // key tiles, and keys in them
  int slot;                // of partial rows, -1: the unit is whole
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
    p.row0 = block * kBlockRows, p.rows = min(kBlockRows, S.count * P.a.group - p.row0);
    const int all = tiles_of(S, P.a.group, block), end = u == ue ? te : all;
    p.tile0 = t, p.n = end - t;
    p.keys = min(end * kKeyTile, keys_of_row(S, P.a.group, p.row0 + p.rows - 1)) - t * kKeyTile;
    p.slot = t == 0 && end == all ? -1 : slot;
    slot = 2 * blockIdx.x + 1;  // (only the first and the last of a block are parts)
    if (end == all) ++u, t = 0;
    else t = end;
    return true;
  }
};

// Values that are no numbers.  In a tile that some rows do not see whole they must not reach those, and 0 times one is none: their groups
// are 0 there, and the rows that see them become none in the end, in these 32 numbers alone.  Which those are, of a row that sees `lim` keys
// and a block's piece `i`, is looked up here by the row's warp, once the block has met such a value: a bit for each group.  (Not inlined: 48
// tokens of 8 sequences 123.8 us, as without; inlined 124.8.)
template <typename T, int kDim, bool kImage>
__device__ __noinline__ uint32_t groups_that_are_none(const PackedTcParams& P, int i, int lim) {
  constexpr int kGroups = kDim / 32;
  Pieces pieces(P);
  Piece U;
  for (int x = 0; x <= i; ++x) pieces.next(P, U);
  const PackedAttnSeq& S = P.a.seq[U.b];
  const uint32_t* ms = reinterpret_cast<const uint32_t*>(P.a.at.scales + P.a.at.scales_v + P.a.at.row0(S.slot, U.hkv) * (kDim / 8));
  const int from = max(keys_of_row(S, P.a.group, kImage ? 0 : U.row0) / kKeyTile, U.tile0) * kKeyTile, to = min((U.tile0 + U.n) * kKeyTile, S.length);
  uint32_t none = 0;
#pragma unroll 1
  for (int g = 0; g < kGroups; ++g) {
    int first = INT_MAX;  // the first key whose group is none
#pragma unroll 1
    for (int j = from + (threadIdx.x & 31); j < to && first == INT_MAX; j += 32)
      if (Codes<T>::odd(__ldg(ms + (int64_t)j * kGroups + g))) first = j;
    __syncwarp();
    first = __reduce_min_sync(0xffffffffu, first);
    if (first < lim) none |= 1u << g;
  }
  return none;
}
}  // namespace xtc

template <typename T, int kDim, bool kImage>
__global__ void __launch_bounds__(xtc::threads(kImage), 1) packed_tc_kernel(const __grid_constant__ PackedTcParams P) {
  using namespace xtc;
  using L = Smem<kDim>;
  constexpr int kWarpMma = kWarpCodes + makers(kImage);
  extern __shared__ __align__(1024) unsigned char smem[];  // (swizzled tiles begin on 1024 bytes, and no byte is left to shift them by)
  const uint32_t s_base = smem_u32(smem), sQ = s_base + L::kQ, sRing = s_base + L::kRing, bars = s_base + L::kBar;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kBar + N_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBar + N_BARS * 8 + 8);
  volatile int* odd_flag = abort_flag + 1;  // a value that is no number has been left out of a tile
  auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* const err = P.a.err;
  if (s_base & 1023) {
    if (threadIdx.x == 0) record_error(err, kErrWaitTimeout, 750);
    return;
  }

  if (warp == 0) {
    static_assert(N_BARS <= 32 && N_BARS * 8 + 16 <= 256, "");
    // tiles: the warps that make them; queries and probabilities: a team's four; what the teams have of the same rows: both
    if (lane < N_BARS) mbar_init(bar(lane), lane < EMPTY0 ? (kImage ? 1u : kCodeWarps / 2u) : lane == Q_FULL0 || lane == Q_FULL0 + 1 || lane == P_FULL0 || lane == P_FULL0 + 1 ? 4u : lane == MERGE ? 8u : 1u);
    if (lane == 0) *abort_flag = 0, *odd_flag = 0;
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
  constexpr uint32_t idesc_qk = make_idesc(kBf16, 128, 128, false), idesc_pv = make_idesc(kBf16, 128, kDim, true);
  chain_enter();

  if (kImage && warp == kWarpCodes) {
    // ========================================================================================================== tiles
    const bool lead = elect_one();
    Pieces pieces(P);
    Piece U;
    bool ok = true;
    int base = 0;
    while (ok && pieces.next(P, U)) {
      const PackedAttnSeq& S = P.a.seq[U.b];
      const char* from = P.image + ((int64_t)S.keys + (int64_t)U.hkv * ((S.length + kKeyTile - 1) / kKeyTile) + U.tile0) * (2 * L::kTileBytes);
      for (int p = 0; p < 2 * U.n && ok; ++p) {
        if (base == 0 && p == min(2 * U.n - 1, kStages - 1)) {  // (behind the first loads, and before a unit's last)
          const int4* odd = reinterpret_cast<const int4*>(P.odd);
          int any = 0;
          for (int x = lane; x < P.n_image / 4; x += 32) any |= odd[x].x | odd[x].y | odd[x].z | odd[x].w;
          for (int x = P.n_image / 4 * 4 + lane; x < P.n_image; x += 32) any |= P.odd[x];
          if (__any_sync(0xffffffffu, any != 0) && lead) *odd_flag = 1;
        }
        const int b = (base + p) % kStages;
        if (base + p >= kStages) ok = warp_wait(bar(EMPTY0 + b), ring_parity(base + p - kStages, kStages), abort_flag, err, 751);
        if (ok && lead) {
          mbar_expect_tx(bar(FULL0 + b), L::kTileBytes);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       ::"r"(sRing + b * L::kTileBytes), "l"(from + (int64_t)(2 * tile_at(p, U.n) + is_value(p, U.n)) * L::kTileBytes), "r"((uint32_t)L::kTileBytes), "r"(bar(FULL0 + b))
                       : "memory");
        }
        __syncwarp();
      }
      if (ok) base += 2 * U.n;
    }
    if (!ok && lane == 0) {  // given up: loads on their way get a bounded chance to land
      for (uint32_t w = 0; w < 4096; ++w) __nanosleep(64);
    }
    __syncwarp();
  } else if (!kImage && warp >= kWarpCodes && warp < kWarpMma) {
    // ======================================================================================================== numbers
    // Half of the warps take key tiles, half value tiles.  A thread has the 32 numbers of one (m, s), a 16-byte piece of a row of codes, of
    // kPer rows; the next tile's are on their way through registers while it is at work, those kAhead tiles ahead to L2.
    // (Eight lanes that write 16 bytes at a time have four rows and pieces of one half of them: eight different bank groups.)
    using C = Codes<T>;
    constexpr int kGroups = kDim / 32, kStep = kCodeWarps / 2 * 32 / kGroups, kPer = (128 + kStep - 1) / kStep, kAhead = 4;
    constexpr int kRow = kDim / 2, kScales = kDim / 8;  // bytes
    static_assert(kStep % 8 == 0, "");
    const bool values = warp >= kWarpCodes + kCodeWarps / 2;
    const int w8 = (warp - kWarpCodes) % (kCodeWarps / 2), at = w8 * 32 + lane;
    const int t = kGroups == 4 ? (lane >> 3 & 1) * 2 + (lane & 1) : lane & 1;
    const int r0 = w8 * (32 / kGroups) + (kGroups == 4 ? (lane >> 4) * 4 + (lane >> 1 & 3) : lane >> 1);
    struct Raw {
      uint32_t c[kPer][4], ms[kPer];
    };
    Pieces pieces(P);
    bool more = false;
    int i = 0, n = 0, base = 0;     // the tile of the piece's, and the piece's place in the ring
    int keys = 0, seen = 0;         // from the tile's first one to the piece's last; of those that every row sees
    const char *codes = nullptr, *scales = nullptr;  // this thread's of the tile's first row
    auto begin = [&]() {
      Piece U;
      more = pieces.next(P, U);
      if (!more) return;
      const PackedAttnSeq& S = P.a.seq[U.b];
      const int64_t row = P.a.at.row0(S.slot, U.hkv) + U.tile0 * kKeyTile;
      base += 2 * n, i = 0, n = U.n, keys = U.keys, seen = keys_of_row(S, P.a.group, U.row0) - U.tile0 * kKeyTile;
      codes = P.a.at.codes + (values ? P.a.at.codes_v : 0) + row * kRow + r0 * kRow + t * 16;
      scales = P.a.at.scales + (values ? P.a.at.scales_v : 0) + row * kScales + r0 * kScales + t * 4;
    };
    auto advance = [&]() {
      if (i + 1 < n) ++i, keys -= kKeyTile, seen -= kKeyTile, codes += kKeyTile * kRow, scales += kKeyTile * kScales;
      else begin();
    };
    // lines of 128 bytes of a tile kAhead tiles on: its codes' and its scales'
    constexpr int kLines = kRow, kAll = kLines + kScales;
    static_assert(kAll <= kCodeWarps / 2 * 32, "");
    const int fetch_key = kAhead * kKeyTile + (at < kLines ? at * 128 / kRow : (at - kLines) * 128 / kScales);
    const int fetch = at < kLines ? (fetch_key - r0) * kRow - t * 16 : (fetch_key - r0) * kScales - t * 4;  // from this thread's own
    auto load = [&](Raw& r) {
      // what lies behind the last key is not read: its numbers are 0 by their (m, s), whatever their codes
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const bool there = more && r0 + x * kStep < min(keys, kKeyTile);
        r.ms[x] = 0;
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %7, 0;\n\t"
                     "@p ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%5];\n\t"
                     "@p ld.global.nc.u32 %4, [%6];\n\t}"
                     : "+r"(r.c[x][0]), "+r"(r.c[x][1]), "+r"(r.c[x][2]), "+r"(r.c[x][3]), "+r"(r.ms[x])
                     : "l"(codes + x * kStep * kRow), "l"(scales + x * kStep * kScales), "r"((int)there));
      }
      if (more && at < kAll && fetch_key < keys) asm volatile("prefetch.global.L2 [%0];" ::"l"((at < kLines ? codes : scales) + fetch));
    };
    uint32_t piece[4];  // of a tile: where this thread's 16 bytes go
#pragma unroll
    for (int j = 0; j < 4; ++j) piece[j] = (t >> 1) * kSubTileBytes + r0 * 128 + ((((t & 1) * 4 + j) ^ (r0 & 7)) << 4);
    // (two copies of a turn, each with its own registers: what is on its way is not to be moved, which would wait for it)
    auto turn = [&](Raw& raw, Raw& then) {
      const int slot = base + (values ? pos_v(i, n) : pos_k(i));
      if (values && seen < kKeyTile) {  // (groups_that_are_none)
        bool any = false;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
          const bool odd = C::odd(raw.ms[x]);
          raw.ms[x] = odd ? 0 : raw.ms[x];
          any = any || odd;
        }
        if (any) *odd_flag = 1;
      }
      advance();
      load(then);
      const int b = slot % kStages;
      // (a tile of the other kind, up to three places before in the ring, has not passed this one: the phase is the next one of the barrier)
      if (slot >= kStages && !warp_wait(bar(EMPTY0 + b), ring_parity(slot - kStages, kStages), abort_flag, err, 751)) return false;
      unsigned char* to = smem + L::kRing + b * L::kTileBytes;
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        if ((x + 1) * kStep > 128 && r0 + x * kStep >= 128) continue;
        const auto m2 = C::least2(raw.ms[x]), s2 = C::step2(raw.ms[x]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w[4];
          C::pairs(raw.c[x][j], m2, s2, w);
          *reinterpret_cast<uint4*>(to + piece[j] + x * kStep * 128) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(FULL0 + b));
      return more;
    };
    Raw raw{}, then{};
    begin();
    load(raw);
    while (more && turn(raw, then) && turn(then, raw)) {
    }
    __syncwarp();
  } else if (warp == kWarpMma) {
    // ===================================================================================================== products
    const bool lead = elect_one();
    int base = 0, np[2] = {0, 0}, n_one = 0, n_two = 0;  // ring position, probabilities that have been waited for, units of each kind
    bool ok = true;
    const uint64_t ring_k = make_sdesc(sRing, 16, 1024), ring_v = make_sdesc(sRing, kSubTileBytes, 1024), qd0 = make_sdesc(sQ, 16, 1024);
    auto arrived = [&](int pos) { ok = ok && warp_wait(bar(FULL0 + pos % kStages), ring_parity(pos, kStages), abort_flag, err, 761); };
    auto release = [&](int pos) {
      if (lead) tc_commit(bar(EMPTY0 + pos % kStages));
    };
    auto qk = [&](int q, int pos, int team) {  // S of a team, of one of the tiles of queries
      tc_fence_after();
      if (lead) {
        const uint64_t qd = qd0 + (uint64_t)(q * L::kTileBytes >> 4), kd = ring_k + (uint64_t)((pos % kStages) * L::kTileBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks) {
          const uint64_t o = (uint64_t)(((ks >> 2) * kSubTileBytes + (ks & 3) * 32) >> 4);
          mma_ss(tmem + team * 128, qd + o, kd + o, idesc_qk, ks > 0);
        }
        tc_commit(bar(S_FULL0 + team));
      }
      __syncwarp();
    };
    auto pv = [&](int team, int pos, bool first) {
      ok = ok && warp_wait(bar(P_FULL0 + team), np[team] & 1, abort_flag, err, 762);
      ++np[team];
      if (!ok) return;
      tc_fence_after();
      if (lead) {
        const uint64_t vd = ring_v + (uint64_t)((pos % kStages) * L::kTileBytes >> 4);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) mma_ts(tmem + 256 + team * 128, tmem + team * 128 + 8 * ks, vd + (uint64_t)((ks * 2048) >> 4), idesc_pv, !first || ks > 0);
        tc_commit(bar(PV_DONE0 + team));
      }
      __syncwarp();
    };
    Pieces pieces(P);
    Piece U;
    while (ok && pieces.next(P, U)) {
      const int n = U.n;
      const bool two = U.rows > 128;
      ok = warp_wait(bar(Q_FULL0), n_one++ & 1, abort_flag, err, 760);
      if (two) ok = ok && warp_wait(bar(Q_FULL0 + 1), n_two++ & 1, abort_flag, err, 760);
      if (!ok) break;
      const int ahead = two ? 1 : 2;  // tiles that both teams, or one after the other, have scores of
      for (int i = 0; i < ahead && i < n && ok; ++i) {
        const int pos = base + pos_k(i);
        arrived(pos);
        if (!ok) break;
        qk(0, pos, two ? 0 : i);
        if (two) qk(1, pos, 1);
        release(pos);
      }
      for (int i = 0; i < n && ok; ++i) {
        const int v_pos = base + pos_v(i, n), more = i + ahead, k_pos = base + pos_k(more);
        arrived(v_pos);
        if (!ok) break;
        if (two) {
          pv(0, v_pos, i == 0);
          if (ok && more < n) {
            arrived(k_pos);
            if (ok) qk(0, k_pos, 0);
          }
          if (ok) pv(1, v_pos, i == 0);
          if (!ok) break;
          release(v_pos);
          if (more < n) {
            qk(1, k_pos, 1);
            release(k_pos);
          }
        } else {
          pv(i & 1, v_pos, i < 2);
          if (!ok) break;
          release(v_pos);
          if (more < n) {
            arrived(k_pos);
            if (!ok) break;
            qk(0, k_pos, i & 1);
            release(k_pos);
          }
        }
      }
      base += 2 * n;
    }
    // Nothing will be signalled in this block when it goes: the releases come behind all products.  (That a tile has been there says that the
    // one before it in its place had been released: the phase waited for is the next one.)
    for (int b = 0; b < kStages && ok; ++b) {
      const int last = ring_last(base, kStages, b);
      if (last >= 0) ok = warp_wait(bar(EMPTY0 + b), ring_parity(last, kStages), abort_flag, err, 752);
    }
    __syncwarp();
  } else if (warp < kWarpCodes) {
    // ====================================================================================================== softmax
    const int quad = warp & 3, team = warp >> 2, row = quad * 32 + lane;
    const uint32_t lane_base = ((uint32_t)(quad * 32)) << 16;
    const uint32_t tO = tmem + 256 + team * 128 + lane_base;
    struct Turn {  // a unit, and this thread's row of it
      bool more, two, in;
      bool idle;  // the warp has no row of it: what it leaves in P is of rows that nobody looks at
      int n, mine, key0, lim, all;  // its tiles; this team's
      int64_t out, slot_row;  // row of the output; of the partial results, -1: the unit is whole
      int64_t part;           // the first of the row's 32 in its slot's numbers
      int64_t lse;            // of the counted rows' log-sum-exps
      int64_t q;              // bytes from the first query's first row to its own, -1: none
    };
    Pieces pieces(P);
    auto find = [&]() {
      Turn t;
      Piece U;
      t.more = pieces.next(P, U);
      if (!t.more) return t;
      const PackedAttnSeq& S = P.a.seq[U.b];
      t.n = U.n, t.key0 = U.tile0 * kKeyTile, t.two = U.rows > 128;
      t.mine = t.two ? t.n : (t.n + 1 - team) / 2;
      const int at = (t.two ? team * 128 : 0) + row;
      t.in = at < U.rows;
      t.lim = t.key0 + U.keys;  // rows that are none are not masked, so that whole tiles stay whole: nothing of them is written
      t.out = t.lse = 0, t.slot_row = t.part = t.q = -1;
      if (t.in) {
        const int r = U.row0 + at, i = r / P.a.group, h = r - i * P.a.group;
        t.lim = min(t.lim, keys_of_row(S, P.a.group, r));
        const int64_t b = P.a.b0 + U.b, tok = P.a.most - S.count + i;
        t.q = b * P.a.q_bs + (int64_t)(U.hkv * P.a.group + h) * P.a.q_hs + tok * P.a.q_ts;
        t.out = (b * P.a.most + tok) * (P.a.at.n_kv * P.a.group) + U.hkv * P.a.group + h;
        t.lse = (b * P.a.at.n_kv + U.hkv) * P.a.most * P.a.group + r;
      }
      if (U.slot >= 0) {
        t.slot_row = (int64_t)U.slot * kBlockRows + at;
        t.part = ((int64_t)U.slot * kBlockRows + at - lane) * kDim;
      }
      t.all = __reduce_min_sync(0xffffffffu, t.lim);
      t.idle = at - lane >= U.rows;
      return t;
    };
    auto queries = [&](const Turn& t) {
      // The warp's 32 rows, 16 bytes a lane, swizzled.  No product reads the last unit's any more: its scores have been seen.
      constexpr int kPer = kDim / 8, kAt = 32 / kPer;
      const int c = lane % kPer;
      const uint32_t to = sQ + team * L::kTileBytes + quad * 32 * 128 + (c >> 3) * kSubTileBytes;
#pragma unroll 1
      for (int r = lane / kPer; r < 32; r += kAt) {
        const int64_t from = __shfl_sync(0xffffffffu, t.q, r);
        mma::cp_async16(to + r * 128 + (((c & 7) ^ (r & 7)) << 4), P.a.q + (from < 0 ? 0 : from) + c * 16, from >= 0);
      }
      mma::cp_async_commit();
      mma::cp_async_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Q_FULL0 + team));
    };
    float2* const ml = reinterpret_cast<float2*>(smem + L::kMl);  // of each team's rows, where both have the same
    int piece = 0;                     // of the block's
    int ns[2] = {0, 0}, n_merged = 0;  // tiles so far of each team; arrivals of both at MERGE
    bool ok = true, owed = false;      // the other team may still read this one's O
    const uint32_t tS = tmem + team * 128 + lane_base;
    Turn now = find();
    if (now.more && (now.two || team == 0)) queries(now);
    while (now.more && ok) {
      const Turn next = find();
      float m = -INFINITY, l = 0.f;
      for (int x = 0; x < now.mine && ok; ++x) {
        const int i = now.two ? x : 2 * x + team;
        ok = warp_wait(bar(S_FULL0 + team), (ns[team] + x) & 1, abort_flag, err, 770);
        if (!ok) break;
        tc_fence_after();
        if (now.idle) {
          if (owed) ok = warp_wait(bar(MERGE), (n_merged - 1) & 1, abort_flag, err, 773), owed = false;
          if (!ok) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(P_FULL0 + team));
          continue;
        }
        const int j0 = now.key0 + i * kKeyTile;
        if (now.all < j0 + kKeyTile) {
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
        const float mt = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]) * P.a.scale_log2;
        const float mn = mt - m > Reference<T>::kGrow ? mt - Reference<T>::kBelow : m;  // (from -inf: any number)
        const float alpha = m == -INFINITY ? 1.f : ex2_approx(m - mn);
        const bool scale_o = __any_sync(0xffffffffu, mn != m && m != -INFINITY) && x > 0;
        l *= alpha;
        m = mn;
        const float nm = m == -INFINITY ? 0.f : -m;
        float2 rs[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // P, packed, takes the place of scores that have been read: 16 columns for 32
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float2 e[16];
          uint32_t pk[16];
          arg_chunk(s, P.a.scale_log2, nm, e);
          tmem_ld32_if(c < 3, tS + 32 * c + 32, us);
          exp_chunk<T, 5>(e, rs, pk);
          tmem_st16(tS + 16 * c, pk);
          tmem_wait_ld32(us);
        }
        const float2 r = fadd2(fadd2(rs[0], rs[1]), fadd2(rs[2], rs[3]));
        l += r.x + r.y;
        if (scale_o) {
          // O has the products up to the tile before: wait for the last of them
          ok = warp_wait(bar(PV_DONE0 + team), (ns[team] + x - 1) & 1, abort_flag, err, 771);
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
        if (owed) ok = warp_wait(bar(MERGE), (n_merged - 1) & 1, abort_flag, err, 773), owed = false;
        if (!ok) break;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL0 + team));
      }
      const bool merge = !now.two && now.n > 1;
      // the next unit's queries first, so that its first scores are formed while this one's rows are written; where both teams
      // have the same queries, once the other one is through with them too
      const bool load = next.more && (next.two || team == 0);
      if (ok && load && !merge) queries(next);
      if (ok && now.mine > 0) ok = warp_wait(bar(PV_DONE0 + team), (ns[team] + now.mine - 1) & 1, abort_flag, err, 772);
      // rows that both teams have a part of: each writes half of their columns
      float mine = 1.f, theirs = 0.f;
      if (ok && merge) {
        ml[team * 128 + row] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(MERGE));
        ok = warp_wait(bar(MERGE), n_merged++ & 1, abort_flag, err, 775);
        if (ok) {
          if (load) queries(next);
          tc_fence_after();
          const float2 o = ml[(team ^ 1) * 128 + row];
          const float mx = fmaxf(m, o.x), ref = mx == -INFINITY ? 0.f : mx;
          mine = exp2f(m - ref), theirs = exp2f(o.x - ref);
          l = l * mine + o.y * theirs;
          m = mx;
        }
      }
      if (ok && (now.two || merge || team == 0)) {
        tc_fence_after();
        const float inv = l > 0.f ? 1.f / l : l;  // (a NaN stays one)
        mine *= inv, theirs *= inv;
        const uint32_t none = __any_sync(0xffffffffu, *odd_flag) ? groups_that_are_none<T, kDim, kImage>(P, piece, now.lim) : 0;
#pragma unroll 1
        for (int c = merge ? team * (kDim / 2) : 0; c < (merge && team == 0 ? kDim / 2 : kDim); c += 32) {
          uint32_t o[32];
          float* f = reinterpret_cast<float*>(o);
          tmem_ld32(tO + c, o);
          tmem_wait_ld32(o);
          const float by = none >> (c / 32) & 1 ? NAN : mine;
#pragma unroll
          for (int k = 0; k < 32; ++k) f[k] *= by;
          if (merge) {
            uint32_t z[32];
            tmem_ld32(tmem + 256 + (team ^ 1) * 128 + lane_base + c, z);
            tmem_wait_ld32(z);
#pragma unroll
            for (int k = 0; k < 32; ++k) f[k] = fmaf(__uint_as_float(z[k]), theirs, f[k]);
          }
          if (now.in && now.slot_row >= 0) {
            // partial rows lie in blocks of 32, four columns of all of them side by side: every store is one stretch
            float4* to = reinterpret_cast<float4*>(P.a.part_o + now.part) + (c / 4) * 32 + lane;
#pragma unroll
            for (int k = 0; k < 8; ++k) to[k * 32] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
          } else if (now.in) {
            uint4* to = reinterpret_cast<uint4*>(P.a.out + (now.out * kDim + c) * 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = mma::pack2<T>(f[8 * k + 2 * e], f[8 * k + 2 * e + 1]);
              to[k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          __syncwarp();
        }
        if (now.in && (now.two || team == 0)) {
          const float lse = l > 0.f ? m + log2f(l) : l == 0.f ? -INFINITY : l;
          if (now.slot_row >= 0) {
            P.a.part_lse[now.slot_row] = lse;
          } else {
            if (P.a.lse) P.a.lse[now.out] = lse * (1.f / kLog2e);
            if (P.a.row_lse) P.a.row_lse[now.lse] = lse;
          }
        }
        tc_fence_before();
      }
      if (ok && merge) {  // both teams' O have been read: no probabilities are handed over before
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(MERGE));
        ++n_merged, owed = true;
      }
      if (now.two) ns[0] += now.n, ns[1] += now.n;
      else ns[0] += (now.n + 1) / 2, ns[1] += now.n / 2;
      __syncwarp();
      now = next, ++piece;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) tmem_dealloc(tmem, 512);
}

// The numbers of all tiles of a launch's sequences, each as a block of the kernel above wants it in its shared memory: for prompts, whose
// tiles many blocks read (2048 tokens behind 28000: 32 blocks of rows).  A tile of keys or of values a block: out of its codes in shared
// memory, and from there in one piece.
template <typename T, int kDim>
__global__ void __launch_bounds__(256) packed_image_kernel(const __grid_constant__ PackedTcParams P) {
  using L = xtc::Smem<kDim>;
  using C = Codes<T>;
  constexpr int kGroups = kDim / 32, kPer = 128 * kGroups / 256;
  extern __shared__ __align__(1024) unsigned char smem[];
  int lo = 0, hi = P.a.batch - 1;
  const int tile = blockIdx.x;
  while (lo < hi) {  // (the sequence's first tile is in `keys`)
    const int mid = (lo + hi + 1) / 2;
    if (P.a.seq[mid].keys <= tile) lo = mid;
    else hi = mid - 1;
  }
  const PackedAttnSeq S = P.a.seq[lo];
  const int tiles = (S.length + kKeyTile - 1) / kKeyTile, hkv = (tile - S.keys) / tiles, j0 = (tile - S.keys) % tiles * kKeyTile;
  const bool mixed = j0 + kKeyTile > keys_of_row(S, P.a.group, 0);
  bool odd = false;
  chain_enter();
  for (int value = 0; value < 2; ++value) {
    const int64_t row = P.a.at.row0(S.slot, hkv) + j0;
    const char* codes = P.a.at.codes + (value ? P.a.at.codes_v : 0) + row * (kDim / 2);
    const char* scales = P.a.at.scales + row * (kDim / 8);
    uint4 c[kPer];
    uint32_t ms[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const int at = threadIdx.x + x * 256, k = at / kGroups, t = at % kGroups;
      c[x] = make_uint4(0, 0, 0, 0), ms[x] = 0;
      if (j0 + k < S.length) {
        c[x] = __ldg(reinterpret_cast<const uint4*>(codes + k * (kDim / 2) + t * 16));
        ms[x] = __ldg(reinterpret_cast<const uint32_t*>(scales + (value ? P.a.at.scales_v : 0) + k * (kDim / 8) + t * 4));
        if (mixed && value && C::odd(ms[x])) ms[x] = 0, odd = true;  // (as the warps that do this without an image)
      }
    }
    if (value) {
      if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // (the keys have been read from where the values go)
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const int at = threadIdx.x + x * 256, k = at / kGroups, t = at % kGroups;
      put_group<T>(smem + (t >> 1) * kSubTileBytes, k, t, c[x], ms[x]);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    const int any = __syncthreads_or(odd);
    if (threadIdx.x == 0) {
      if (value) P.odd[tile] = any;
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(P.image + ((int64_t)2 * tile + value) * L::kTileBytes), "r"(smem_u32(smem)), "r"((uint32_t)L::kTileBytes) : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

template <typename T, int kDim, bool kImage>
static int tc_launch(const PackedTcParams& P, cudaStream_t s) {
  auto kern = packed_tc_kernel<T, kDim, kImage>;
  const int smem = xtc::Smem<kDim>::kTotal;
  static std::atomic<uint64_t> set;  // devices that know it
  int dev = 0;
  INFLLM_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !(set.load(std::memory_order_relaxed) >> dev & 1)) {
    INFLLM_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev < 64) set.fetch_or(1ull << dev);
  }
  if (kImage) {
    INFLLM_CUDA_OK(launch_chained(packed_image_kernel<T, kDim>, dim3(P.n_image), dim3(256), xtc::Smem<kDim>::kTileBytes, s, P));
    INFLLM_LAUNCH_OK("packed_image_kernel");
  }
  INFLLM_CUDA_OK(launch_chained(kern, dim3(P.n_ctas), dim3(xtc::threads(kImage)), smem, s, P));
  INFLLM_LAUNCH_OK("packed_tc_kernel");
  return INFLLM_OK;
}

int packed_tc_launch(const PackedTcParams& P, int dtype, int head_dim, cudaStream_t s) {
  INFLLM_DISPATCH_DTYPE(dtype, T, {
    if (P.image) return head_dim == 128 ? tc_launch<T, 128, true>(P, s) : tc_launch<T, 64, true>(P, s);
    return head_dim == 128 ? tc_launch<T, 128, false>(P, s) : tc_launch<T, 64, false>(P, s);
  });
}

}  // namespace infllm
