// The cache in 4 bits (packed.cuh has the format): writes, reads, and eviction by attention weight.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "packed.cuh"

namespace infllm {

namespace cg = cooperative_groups;

constexpr int kPackSeqs = 128;  // of a launch

// ------------------------------------------------------------------------------------------------------------ writes
constexpr int kPackThreads = 128;

struct PackWriteParams {
  const char *k, *v, *q;
  char* q_out;                                                   // (B, L, n_heads, dim)
  int64_t k_bs, k_hs, k_ts, v_bs, v_hs, v_ts, q_bs, q_hs, q_ts;  // bytes
  PackedPlanes at;
  float* weights;
  int32_t* places;
  const float *cos_t, *sin_t;                                    // null: nothing is rotated
  int32_t n_heads, most, b0, tokens, per_block;                  // tokens of the launch, and of a block
  PackedSeq seq[kPackSeqs];
};

// the least and the largest of a group, whose 32 numbers four neighbouring threads have; NaN if one of them is
template <typename T>
__device__ __forceinline__ float2 span32(const uint4& x, uint32_t quad) {
  using T2 = typename Act<T>::T2;
  const T2* p = reinterpret_cast<const T2*>(&x);
  const T2 lo = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3]));
  const T2 hi = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
  T2 ends = {__hmin_nan(lo.x, lo.y), __hneg(__hmax_nan(hi.x, hi.y))};  // (the largest as the least of the negatives)
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) ends = __hmin2_nan(ends, __shfl_xor_sync(quad, ends, o));
  return make_float2(Act<T>::to_f(ends.x), -Act<T>::to_f(ends.y));
}

// a span's fifteenth, rounded once (below, its second term would be rounded to fewer bits)
__device__ __forceinline__ float fifteenth(float span) {
  constexpr float kHi = 1.f / 15.f, kLo = (float)(1. / 15. - (double)kHi);
  return span < 0x1p-90f ? __fdiv_rn(span, 15.f) : fmaf(span, kHi, span * kLo);
}
// Eight numbers of a row as codes, and their group's (m, s).
// A quotient of 16-bit numbers' differences lies on the border between two codes, or further from it than the last place in 32 bits: so
// a rounded quotient has the definition's code.  1 / s as the sum of two numbers, of which the second is what the first leaves (1 - inv s is
// exact), is right to 2^-46; so t inv + t rest, rounded once, is the border wherever the quotient is one: three operations a number, with the
// rounding to a whole one, instead of a division's dozen.  Steps at the ends of the range, where the reciprocal or what it leaves is
// no normal number, or fp16's steps of less than 16 of its least ones, where a quotient may be above 15.5, are divided by.
template <typename T>
__device__ __forceinline__ uint32_t pack8(const uint4& x, uint32_t quad, uint32_t* ms) {
  const float2 span = span32<T>(x, quad);
  T step = Act<T>::from_f(fifteenth(span.y - span.x));
  const T least = Act<T>::from_f(span.x);
  float s = Act<T>::to_f(step);
  // m + 15 s is 16 or more above the largest number, 65504, only where s was rounded up by more than 1, so from 4096 on.  (bf16: the largest
  // s that is held, just below 2^122, is rounded by too little.)
  if constexpr (!Codes<T>::kBf16) {
    if (s >= 4096.f && __hisinf(__hfma(step, __float2half(15.f), least)) && !__hisinf(step)) step = __ushort_as_half(__half_as_ushort(step) - 1), s = Act<T>::to_f(step);
  }
  const bool held = s < (Codes<T>::kBf16 ? 0x1p122f : INFINITY);  // (not where one is not finite, either)
  if (!held) step = Act<T>::from_f(NAN);
  const typename Act<T>::T2 pair = {least, step};
  *ms = *reinterpret_cast<const uint32_t*>(&pair);
  const typename Act<T>::T2* p = reinterpret_cast<const typename Act<T>::T2*>(&x);
  uint32_t w = 0;
  if (!held) return 0;
  if (s < (Codes<T>::kBf16 ? 0x1p-100f : 0x1p-20f) || s > 0x1p90f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = Act<T>::to_f2(p[i >> 1]);
      const int c = s == 0.f ? 0 : __float2int_rn(__fdiv_rn((i & 1 ? f.y : f.x) - span.x, s));
      w |= (uint32_t)min(max(c, 0), 15) << (4 * (i >> 1) + 16 * (i & 1));
    }
    return w;
  }
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  const float rest = fmaf(-inv, s, 1.f) * inv;
  constexpr float kMagic = 8388608.f;  // 2^23: what is added to it is rounded to a whole number, ties to even, in its low bits
  constexpr uint32_t kMagicBits = 0x4b000000u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = Act<T>::to_f2(p[i >> 1]);
    const float t = (i & 1 ? f.y : f.x) - span.x, q = fmaf(t, inv, t * rest);
    w += (__float_as_uint(q + kMagic) - kMagicBits) << (4 * (i >> 1) + 16 * (i & 1));
  }
  return w;
}

template <typename T>
__device__ __forceinline__ void pack_rotate8(uint4& lo, uint4& hi, const float* cs, const float* sn) {
  T *a = reinterpret_cast<T*>(&lo), *b = reinterpret_cast<T*>(&hi);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // each product rounded to fp32 first, and the sum to 16 bits: as the rotary embedding of the other attention types
    const float x1 = Act<T>::to_f(a[i]), x2 = Act<T>::to_f(b[i]);
    a[i] = Act<T>::from_f(__fadd_rn(__fmul_rn(x1, cs[i]), __fmul_rn(-x2, sn[i])));
    b[i] = Act<T>::from_f(__fadd_rn(__fmul_rn(x2, cs[i]), __fmul_rn(x1, sn[i])));
  }
}

// A thread has 8 numbers of the first half of a row and the 8 that are rotated with them; the four threads of a group of 32 agree on
// its least number and step.
// What bounds it: bytes, and the arithmetic of codes and angles beside them.  8192 tokens of 32 query and 32 KV heads of 128 in fp16, 310 MB in
// and out: 73 us, 4.2 TB/s, in a row of calls; 63 without angles, 60 with no arithmetic for the codes.  From 85: three operations a number
// instead of five, 83; one exchange for both ends of a group, and no division for the step, 80; the next row ahead, 75; eight blocks a
// multiprocessor, 73 (ten: 77; blocks of 256: 96, of 64: 73).  Of 64 single tokens, 3.6 us.
template <typename T, int kDim, bool kRope>
__global__ void __launch_bounds__(kPackThreads, 8) packed_write_kernel(const __grid_constant__ PackWriteParams P) {
  constexpr int kPer = kDim / 16;  // threads of a row
  const int n_kv = P.at.n_kv, n_rows = P.n_heads + 2 * n_kv, per = min(n_rows * kPer, kPackThreads);  // threads of a token
  const int sub = (int)threadIdx.x / per, of_token = (int)threadIdx.x - sub * per, token = (int)blockIdx.x * P.per_block + sub;
  if (sub >= P.per_block || token >= P.tokens) return;
  const int b = token / P.most, i = token - b * P.most;
  const PackedSeq S = P.seq[b];
  const int at = i - (P.most - S.count);  // of the new tokens (the shorter sequences' stand at the end)
  const int c = of_token % kPer;
  const int64_t bb = P.b0 + b;
  const uint32_t quad = 0xfu << (threadIdx.x & 28);
  float cs[8], sn[8];
  if (kRope && at >= 0) {
    const int64_t o = (int64_t)(S.position + at) * (kDim / 2) + c * 8;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      *reinterpret_cast<float4*>(cs + k) = __ldg(reinterpret_cast<const float4*>(P.cos_t + o + k));
      *reinterpret_cast<float4*>(sn + k) = __ldg(reinterpret_cast<const float4*>(P.sin_t + o + k));
    }
  }
  // (the next row is on its way while one is worked on)
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo, lo1 = lo, hi1 = lo;  // (no token: its query is not one)
  auto load = [&](int r, uint4& a, uint4& z) {
    if (at < 0 || r >= n_rows) return;
    const char* src = r < P.n_heads          ? P.q + bb * P.q_bs + r * P.q_hs + i * P.q_ts
                      : r < P.n_heads + n_kv ? P.k + bb * P.k_bs + (r - P.n_heads) * P.k_hs + i * P.k_ts
                                             : P.v + bb * P.v_bs + (r - P.n_heads - n_kv) * P.v_hs + i * P.v_ts;
    a = *reinterpret_cast<const uint4*>(src + c * 16), z = *reinterpret_cast<const uint4*>(src + kDim + c * 16);
  };
  load(of_token / kPer, lo1, hi1);
  for (int r = of_token / kPer; r < n_rows; r += per / kPer) {
    const bool val = r >= P.n_heads + n_kv;
    const int h = r - P.n_heads - (val ? n_kv : 0);
    if (h >= 0 && at < 0) return;  // (queries come first: nothing is left of this token)
    lo = lo1, hi = hi1;
    load(r + per / kPer, lo1, hi1);
    if (kRope && !val && at >= 0) pack_rotate8<T>(lo, hi, cs, sn);
    if (h < 0) {
      char* to = P.q_out + ((bb * P.most + i) * P.n_heads + r) * (int64_t)(kDim * 2);
      *reinterpret_cast<uint4*>(to + c * 16) = lo;
      *reinterpret_cast<uint4*>(to + kDim + c * 16) = hi;
      continue;
    }
    const int64_t row = P.at.row0(S.slot, h) + S.length - S.count + at;
    uint32_t ms[2];
    const uint32_t w0 = pack8<T>(lo, quad, ms), w1 = pack8<T>(hi, quad, ms + 1);
    uint32_t* codes = reinterpret_cast<uint32_t*>(const_cast<char*>(P.at.codes) + (val ? P.at.codes_v : 0) + row * (kDim / 2));
    uint32_t* scales = reinterpret_cast<uint32_t*>(const_cast<char*>(P.at.scales) + (val ? P.at.scales_v : 0) + row * (kDim / 8));
    codes[c] = w0, codes[kPer + c] = w1;
    if (c % 4 == 0) scales[c / 4] = ms[0], scales[kPer / 4 + c / 4] = ms[1];
    if (!val && c == 0) P.weights[row] = 0.f, P.places[row] = S.position + at;
  }
}

// ------------------------------------------------------------------------------------------------------------- reads
struct PackReadParams {
  char *k, *v;        // (layers, batch, n_kv, most, dim)
  PackedPlanes at;    // of the first layer
  int64_t codes_layer, scales_layer;  // bytes from layer to layer
  int32_t most, b0, batch;
  PackedSeq seq[kPackSeqs];
};

// kReadEach words of eight numbers a thread, of a head's tokens: their loads are all on their way before the first is used.
// What bounds it: the numbers' bytes, 16 bits for 5 bits read.  8192 tokens of 32 heads of 128, keys and values: 176 MB in 29 us, 6.0 TB/s.
constexpr int kReadThreads = 256, kReadEach = 4;
template <typename T, int kDim>
__global__ void __launch_bounds__(kReadThreads) packed_values_kernel(const __grid_constant__ PackReadParams P) {
  constexpr int kWords = kDim / 8;
  const int per = (P.most * kWords + kReadThreads * kReadEach - 1) / (kReadThreads * kReadEach), h = blockIdx.x / per;
  const int first = (blockIdx.x - h * per) * kReadThreads * kReadEach + threadIdx.x, words = P.most * kWords;
  const int layer = blockIdx.z >> 1, val = blockIdx.z & 1;
  const PackedSeq S = P.seq[blockIdx.y];
  const int64_t row0 = P.at.row0(S.slot, h) + S.length - P.most;  // (the tokens stand at the end)
  const char* codes = P.at.codes + layer * P.codes_layer + val * P.at.codes_v;
  const char* scales = P.at.scales + layer * P.scales_layer + val * P.at.scales_v;
  uint4* to = reinterpret_cast<uint4*>(val ? P.v : P.k) + (((int64_t)layer * P.batch + P.b0 + blockIdx.y) * P.at.n_kv + h) * (int64_t)words;
  uint32_t c[kReadEach], ms[kReadEach];
#pragma unroll
  for (int x = 0; x < kReadEach; ++x) {
    const int at = first + x * kReadThreads, i = at / kWords, w = at % kWords;
    c[x] = ms[x] = 0;  // (numbers of no token: 0)
    if (at < words && i >= P.most - S.count) {
      c[x] = __ldg(reinterpret_cast<const uint32_t*>(codes + (row0 + i) * (kDim / 2)) + w);
      ms[x] = __ldg(reinterpret_cast<const uint32_t*>(scales + (row0 + i) * (kDim / 8)) + w / 4);
    }
  }
#pragma unroll
  for (int x = 0; x < kReadEach; ++x) {
    const int at = first + x * kReadThreads;
    uint32_t v[4];
    Codes<T>::pairs(c[x], Codes<T>::least2(ms[x]), Codes<T>::step2(ms[x]), v);
    if (at < words) to[at] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// ---------------------------------------------------------------------------------------------------------- eviction
// Of a head's n tokens the first `sink`, the newest `recent` and the k of largest weight between them stay.  A cluster of blocks
// has a head: the k-th largest weight by its digits of 8 bits from the top (four passes over the weights, whose counts the blocks
// add up through each other's shared memory: with digits of 11 bits that takes longer than the pass that they spare), then each block lists which of its share of tokens stay, at the rank that the
// counts before it give; ties go to the earlier token.  Then the rows close up: a row's new place is never behind its old one,
// so, in place, the blocks read kRound rows each, wait for each other, and write; what the next round reads lies behind all that
// this one has written.
// What bounds it: bytes, where sequences and layers are many (4 sequences of 2176 tokens, 32 layers, 8 KV heads of 128, 2048 stay: 705 MB
// in and out, 140 us into other places, 5.0 TB/s, 116 in place); otherwise the chain of passes, lists and rows, some 15 us (8 sequences of
// 4224, 2 layers, 2048 stay: 86 MB, 29 us; one of 65536, 4 layers, 4096 stay: 50 MB, 34 us, 38 with weights one by one and one count).
constexpr int kEvictThreads = 256, kRound = 256, kEach = 8;
constexpr int kEvictRoom = 10240;  // weights a block: 40 KB, so that four blocks have room on a multiprocessor
constexpr int kCounts = 4, kPitch = 256 + 8;  // counts of a digit, by lanes: weights of like size have few first digits, and wait for each other

struct EvictParams {
  PackedPlanes at;
  int64_t codes_layer, scales_layer;  // bytes
  float* weights;
  int32_t* places;
  int64_t rows_layer;
  int32_t* stay;      // (layers, sequences, KV heads, most_stay): of the middle tokens those that stay
  int64_t seq0, n_seqs, most_stay;
  int32_t budget, sink, recent, room;  // weights that shared memory has room for
  bool copy;
  int2 seq[kPackSeqs];   // slot, length
  int32_t into[kPackSeqs];
};

// whole numbers in the order of the weights
__device__ __forceinline__ uint32_t weight_rank(float w) {
  const uint32_t b = __float_as_uint(w + 0.f);  // (-0 is 0)
  return w != w ? 0xffffffffu : b >> 31 ? ~b : b | 0x80000000u;
}

template <int kDim>
__global__ void __launch_bounds__(kEvictThreads, 4) packed_evict_kernel(const __grid_constant__ EvictParams P) {
  cg::cluster_group cluster = cg::this_cluster();
  const int n_ctas = (int)cluster.num_blocks(), me = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x / n_ctas, b = blockIdx.y, layer = blockIdx.z;
  const int slot = P.seq[b].x, n = P.seq[b].y;
  if (n <= P.budget && !P.copy) return;  // (the whole cluster)
  const bool all = n <= P.budget;
  const int kept = all ? n : P.budget, sink = all ? n : P.sink, late = n - P.recent, k = P.budget - P.sink - P.recent;
  const int64_t from = P.at.row0(slot, h), to = P.copy ? P.at.row0(P.into[b], h) : from;
  const float* weights = P.weights + layer * P.rows_layer + from;
  int32_t* stay = P.stay + (((int64_t)layer * P.n_seqs + P.seq0 + b) * P.at.n_kv + h) * P.most_stay;
  __shared__ int hist[2][256], part[kCounts][kPitch], total[kEvictThreads / 32], counts[2], warps[2][kEvictThreads / 32], found[2], src[kRound];

  const bool choose = !all && k > 0;
  if (choose) {
    const int share = (late - sink + n_ctas - 1) / n_ctas, first = sink + min(me * share, late - sink), last = min(first + share, late);
    // The share's weights, as whole numbers, in shared memory as far as there is room, up to a multiple of 8 with zeros, which are less than
    // any weight's; the others are read again each time
    extern __shared__ __align__(16) uint32_t ranks[];
    const int held = min(last - first, P.room), beyond = first + held;
#pragma unroll 8
    for (int j = tid; j < held; j += kEvictThreads) ranks[j] = weight_rank(weights[first + j]);
    if (tid < (-held & 7)) ranks[held + tid] = 0;
    auto each = [&](auto&& f) {
#pragma unroll 2
      for (int v = tid; v < (held + 3) / 4; v += kEvictThreads) {
        const uint4 u = reinterpret_cast<const uint4*>(ranks)[v];
        f(u.x), f(u.y), f(u.z), f(u.w);
      }
      for (int j = beyond + tid; j < last; j += kEvictThreads) f(weight_rank(weights[j]));
    };
    uint32_t cut = 0;
    int need = k;
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      int* mine = hist[pass & 1];
#pragma unroll
      for (int x = 0; x < kCounts; ++x) part[x][tid] = 0;
      __syncthreads();
      each([&](uint32_t u) {
        if (pass == 0 || (u ^ cut) >> (shift + 8) == 0) atomicAdd(&part[lane % kCounts][u >> shift & 255], 1);
      });
      __syncthreads();
      mine[tid] = part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
      cluster.sync();  // (of the pass after the next, whose counts take this one's place, nobody is ahead of the next one's)
      int sum = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c)  // (all on their way at once)
        if (c < n_ctas) sum += cluster.map_shared_rank(mine, c)[255 - tid];
      // digits from the largest down: how many tokens have a larger one
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      if (lane == 31) total[warp] = upto;
      __syncthreads();
      for (int w = 0; w < warp; ++w) upto += total[w];
      if (upto >= need && upto - sum < need) found[0] = 255 - tid, found[1] = upto - sum;
      __syncthreads();
      cut |= (uint32_t)found[0] << shift;
      need -= found[1];
    }
    // of the tokens of weight `cut` the first `need` stay
    int larger = 0, equal = 0;
    each([&](uint32_t u) { larger += u > cut, equal += u == cut; });
    larger = __reduce_add_sync(0xffffffffu, larger), equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) warps[0][warp] = larger, warps[1][warp] = equal;
    __syncthreads();
    if (tid < 2) {
      int sum = 0;
      for (int w = 0; w < kEvictThreads / 32; ++w) sum += warps[tid][w];
      counts[tid] = sum;
    }
    cluster.sync();
    int before_larger = 0, before_equal = 0;
    for (int c = 0; c < me; ++c) {
      const int* theirs = cluster.map_shared_rank(counts, c);
      before_larger += theirs[0], before_equal += theirs[1];
    }
#pragma unroll 1
    for (int base = first; base < last; base += kEvictThreads * kEach) {
      const int j0 = base + tid * kEach;
      alignas(16) uint32_t u[kEach];
      int g = 0, e = 0;
      const int at = j0 - first;
      if (at + kEach <= ((held + 7) & ~7)) {
        *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(ranks + at);
        *reinterpret_cast<uint4*>(u + 4) = *reinterpret_cast<const uint4*>(ranks + at + 4);
      } else {
#pragma unroll
        for (int x = 0; x < kEach; ++x) u[x] = j0 + x < last ? weight_rank(weights[j0 + x]) : 0;
      }
#pragma unroll
      for (int x = 0; x < kEach; ++x) {
        const bool in = j0 + x < last;
        g += in && u[x] > cut, e += in && u[x] == cut;
      }
      int sg = g, se = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sg, o), y = __shfl_up_sync(0xffffffffu, se, o);
        if (lane >= o) sg += x, se += y;
      }
      __syncthreads();
      if (lane == 31) warps[0][warp] = sg, warps[1][warp] = se;
      __syncthreads();
      int at_g = before_larger + sg - g, at_e = before_equal + se - e;
      for (int w = 0; w < kEvictThreads / 32; ++w) {
        if (w < warp) at_g += warps[0][w], at_e += warps[1][w];
        before_larger += warps[0][w], before_equal += warps[1][w];
      }
#pragma unroll
      for (int x = 0; x < kEach; ++x) {
        if (j0 + x >= last) break;
        const bool more = u[x] > cut, same = u[x] == cut;
        if (more || (same && at_e < need)) stay[at_g + min(at_e, need)] = j0 + x;
        at_g += more, at_e += same;
      }
    }
    cluster.sync();  // the list is there, and nobody reads another block's shared memory any more
  }

  // ---- the rows close up
  constexpr int kCode = kDim / 32, kPer = kRound * kCode / kEvictThreads;  // 16-byte pieces of a row's codes; of a thread
  using Scale = typename std::conditional<kDim == 128, uint4, uint2>::type;
  static_assert(kRound == kEvictThreads, "");
  const char* codes = P.at.codes + layer * P.codes_layer;
  const char* scales = P.at.scales + layer * P.scales_layer;
  int32_t* words[2] = {P.places + layer * P.rows_layer, reinterpret_cast<int32_t*>(P.weights) + layer * P.rows_layer};
  const int tail = all ? n : P.budget - P.recent;  // the first of the newest
#pragma unroll 1
  for (int base = P.copy ? 0 : sink; base < kept; base += n_ctas * kRound) {
    const int r0 = base + me * kRound, rows = min(kRound, kept - r0);
    __syncthreads();
    if (tid < rows) src[tid] = r0 + tid < sink ? r0 + tid : r0 + tid < tail ? stay[r0 + tid - sink] : late + r0 + tid - tail;
    __syncthreads();
    uint4 c[2][kPer];
    Scale s[2];
    int32_t word[2];
    // (a row that stays where it is is not touched)
    auto moves = [&](int r) { return r < rows && (P.copy || src[r] != r0 + r); };
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const int r = (tid + x * kEvictThreads) / kCode, p = (tid + x * kEvictThreads) % kCode;
      if (moves(r)) {
#pragma unroll
        for (int v = 0; v < 2; ++v) c[v][x] = *reinterpret_cast<const uint4*>(codes + v * P.at.codes_v + (from + src[r]) * (kDim / 2) + p * 16);
      }
    }
    if (moves(tid)) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        s[v] = *reinterpret_cast<const Scale*>(scales + v * P.at.scales_v + (from + src[tid]) * (kDim / 8));
        word[v] = words[v][from + src[tid]];
      }
    }
    if (!P.copy) cluster.sync();
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const int r = (tid + x * kEvictThreads) / kCode, p = (tid + x * kEvictThreads) % kCode;
      if (moves(r)) {
#pragma unroll
        for (int v = 0; v < 2; ++v) *reinterpret_cast<uint4*>(const_cast<char*>(codes) + v * P.at.codes_v + (to + r0 + r) * (kDim / 2) + p * 16) = c[v][x];
      }
    }
    if (moves(tid)) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        *reinterpret_cast<Scale*>(const_cast<char*>(scales) + v * P.at.scales_v + (to + r0 + tid) * (kDim / 8)) = s[v];
        words[v][to + r0 + tid] = word[v];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------- checks
int packed_check(const infllm_packed* c, const char* what) {
  if (!c) return fail(INFLLM_E_BADARG, "%s: null pointer", what);
  if (c->n_layers < 1 || c->n_kv_heads < 1 || c->n_sequences < 1 || c->max_tokens < 1)
    return fail(INFLLM_E_BADARG, "%s: %d layers, %d KV heads, %d sequences of %d tokens", what, c->n_layers, c->n_kv_heads, c->n_sequences, c->max_tokens);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(INFLLM_E_UNSUPPORTED, "%s: head_dim %d (64 and 128 are built)", what, c->head_dim);
  if (c->dtype != INFLLM_BF16 && c->dtype != INFLLM_FP16) return fail(INFLLM_E_UNSUPPORTED, "dtype code %d", c->dtype);
  if (c->max_tokens > 1 << 28 || c->n_layers > 16384 || c->n_kv_heads > 8192)
    return fail(INFLLM_E_BADARG, "%s: %d layers of %d KV heads, %d tokens (up to 16384, 8192 and 2^28)", what, c->n_layers, c->n_kv_heads, c->max_tokens);
  if (!c->d_codes || !c->d_scales || !c->d_weights || !c->d_places ||
      ((uintptr_t)c->d_codes | (uintptr_t)c->d_scales | (uintptr_t)c->d_weights | (uintptr_t)c->d_places) % 16)
    return fail(INFLLM_E_BADARG, "%s: the cache's memory has to be 16-byte aligned", what);
  return INFLLM_OK;
}

int packed_check_seqs(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int most, const char* what) {
  if (n < 0 || (n > 0 && !seqs)) return fail(INFLLM_E_BADARG, "%s: %d sequences", what, n);
  if (most < 0 || most > c->max_tokens) return fail(INFLLM_E_BADARG, "%s: tensors of %d tokens", what, most);
  for (int i = 0; i < n; ++i) {
    const infllm_packed_seq& s = seqs[i];
    if (s.slot < 0 || s.slot >= c->n_sequences) return fail(INFLLM_E_BADARG, "%s: sequence %d of %d", what, s.slot, c->n_sequences);
    if (s.length < 0 || s.length > c->max_tokens || s.count < 0 || s.count > s.length || s.count > most || s.position < 0 || s.position > INT_MAX - s.count)
      return fail(INFLLM_E_BADARG, "%s: sequence %d: %d tokens, %d new ones from position %d, tensors of %d", what, s.slot, s.length, s.count, s.position, most);
  }
  std::vector<int32_t> slots(n);
  for (int i = 0; i < n; ++i) slots[i] = seqs[i].slot;
  std::sort(slots.begin(), slots.end());
  for (int i = 1; i < n; ++i)
    if (slots[i] == slots[i - 1]) return fail(INFLLM_E_BADARG, "%s: sequence %d twice", what, slots[i]);
  return INFLLM_OK;
}

PackedPlanes packed_planes(const infllm_packed* c, int layer) {
  const int64_t plane = packed_rows(c);
  PackedPlanes p;
  p.codes_v = plane * (c->head_dim / 2), p.scales_v = plane * (c->head_dim / 8);
  p.codes = (const char*)c->d_codes + 2 * layer * p.codes_v, p.scales = (const char*)c->d_scales + 2 * layer * p.scales_v;
  p.max_tokens = c->max_tokens, p.n_kv = c->n_kv_heads;
  return p;
}

}  // namespace infllm

using namespace infllm;

extern "C" int infllm_packed_write(const infllm_packed* c, int layer, const infllm_packed_seq* seqs, int n, int most, const void* d_k,
                                   int64_t k_bs, int64_t k_hs, int64_t k_ts, const void* d_v, int64_t v_bs, int64_t v_hs, int64_t v_ts,
                                   const void* d_q, int64_t q_bs, int64_t q_hs, int64_t q_ts, void* d_q_out, int n_heads,
                                   const float* d_cos, const float* d_sin, int64_t table_len, void* stream) {
  return guarded("packed_write", [&]() -> int {
    INFLLM_TRY(packed_check(c, "packed_write"));
    INFLLM_TRY(packed_check_seqs(c, seqs, n, most, "packed_write"));
    if (layer < 0 || layer >= c->n_layers) return fail(INFLLM_E_BADARG, "packed_write: layer %d of %d", layer, c->n_layers);
    if (n == 0 || most == 0) return INFLLM_OK;
    if (!d_k || !d_v || (d_q && (!d_q_out || n_heads < 1)) || (!d_cos) != (!d_sin)) return fail(INFLLM_E_BADARG, "packed_write: null pointer");
    if (((uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_q | (uintptr_t)d_q_out | (uintptr_t)d_cos | (uintptr_t)d_sin) % 16 ||
        (k_bs | k_hs | k_ts | v_bs | v_hs | v_ts | q_bs | q_hs | q_ts) % 8)
      return fail(INFLLM_E_BADARG, "packed_write: rows must be 16-byte aligned");
    for (int i = 0; i < n; ++i)
      if (d_cos && seqs[i].count > 0 && (int64_t)seqs[i].position + seqs[i].count > table_len)
        return fail(INFLLM_E_BADARG, "packed_write: a rotary table of %lld rows, position %lld", (long long)table_len, (long long)seqs[i].position + seqs[i].count - 1);
    if (d_q && n_heads > 1 << 16) return fail(INFLLM_E_BADARG, "packed_write: %d heads", n_heads);
    if ((int64_t)kPackSeqs * most > INT_MAX && (int64_t)n * most > INT_MAX) return fail(INFLLM_E_BADARG, "packed_write: %lld tokens", (long long)n * most);
    DeviceScope scope(c->device);
    PackWriteParams P;
    P.k = (const char*)d_k, P.v = (const char*)d_v, P.q = (const char*)d_q, P.q_out = (char*)d_q_out;
    P.k_bs = k_bs * 2, P.k_hs = k_hs * 2, P.k_ts = k_ts * 2;
    P.v_bs = v_bs * 2, P.v_hs = v_hs * 2, P.v_ts = v_ts * 2;
    P.q_bs = q_bs * 2, P.q_hs = q_hs * 2, P.q_ts = q_ts * 2;
    P.at = packed_planes(c, layer);
    P.weights = c->d_weights + layer * packed_rows(c), P.places = c->d_places + layer * packed_rows(c);
    P.cos_t = d_cos, P.sin_t = d_sin;
    P.n_heads = d_q ? n_heads : 0, P.most = most;
    P.per_block = std::max(1, kPackThreads / ((P.n_heads + 2 * c->n_kv_heads) * (c->head_dim / 16)));
    for (P.b0 = 0; P.b0 < n; P.b0 += kPackSeqs) {
      const int m = std::min(n - P.b0, kPackSeqs);
      for (int i = 0; i < m; ++i) P.seq[i] = {seqs[P.b0 + i].slot, seqs[P.b0 + i].length, seqs[P.b0 + i].count, seqs[P.b0 + i].position};
      P.tokens = m * most;
      INFLLM_DISPATCH_DTYPE(c->dtype, T, {
        auto kern = c->head_dim == 128 ? (d_cos ? packed_write_kernel<T, 128, true> : packed_write_kernel<T, 128, false>)
                                       : (d_cos ? packed_write_kernel<T, 64, true> : packed_write_kernel<T, 64, false>);
        kern<<<(unsigned)ceil_div(P.tokens, P.per_block), kPackThreads, 0, (cudaStream_t)stream>>>(P);
      });
      INFLLM_LAUNCH_OK("packed_write_kernel");
    }
    return INFLLM_OK;
  });
}

extern "C" int infllm_packed_values(const infllm_packed* c, int layer, int n_layers, const infllm_packed_seq* seqs, int n, int most,
                                    void* d_k, void* d_v, void* stream) {
  return guarded("packed_values", [&]() -> int {
    INFLLM_TRY(packed_check(c, "packed_values"));
    INFLLM_TRY(packed_check_seqs(c, seqs, n, most, "packed_values"));
    if (layer < 0 || n_layers < 1 || layer > c->n_layers - n_layers) return fail(INFLLM_E_BADARG, "packed_values: layers %d and %d more of %d", layer, n_layers - 1, c->n_layers);
    if (n == 0 || most == 0) return INFLLM_OK;
    if (!d_k || !d_v || ((uintptr_t)d_k | (uintptr_t)d_v) % 16) return fail(INFLLM_E_BADARG, "packed_values: the outputs have to be 16-byte aligned");
    const int64_t words = (int64_t)most * (c->head_dim / 8), blocks = c->n_kv_heads * ceil_div(words, kReadThreads * kReadEach);
    if (blocks > INT_MAX || words > INT_MAX - kReadThreads * kReadEach) return fail(INFLLM_E_BADARG, "packed_values: %d tokens of %d KV heads", most, c->n_kv_heads);
    DeviceScope scope(c->device);
    PackReadParams P;
    P.k = (char*)d_k, P.v = (char*)d_v;
    P.at = packed_planes(c, layer);
    P.codes_layer = 2 * P.at.codes_v, P.scales_layer = 2 * P.at.scales_v;
    P.most = most, P.batch = n;
    for (P.b0 = 0; P.b0 < n; P.b0 += kPackSeqs) {
      const int m = std::min(n - P.b0, kPackSeqs);
      for (int i = 0; i < m; ++i) P.seq[i] = {seqs[P.b0 + i].slot, seqs[P.b0 + i].length, seqs[P.b0 + i].count, seqs[P.b0 + i].position};
      const dim3 grid((unsigned)blocks, m, 2 * n_layers);
      INFLLM_DISPATCH_DTYPE(c->dtype, T, {
        auto kern = c->head_dim == 128 ? packed_values_kernel<T, 128> : packed_values_kernel<T, 64>;
        kern<<<grid, kReadThreads, 0, (cudaStream_t)stream>>>(P);
      });
      INFLLM_LAUNCH_OK("packed_values_kernel");
    }
    return INFLLM_OK;
  });
}

extern "C" int infllm_packed_evict(const infllm_packed* c, const infllm_packed_seq* seqs, int n, const int32_t* into, int64_t budget,
                                   int64_t sink, int64_t recent, void* d_work, int64_t work_bytes, void* stream) {
  return guarded("packed_evict", [&]() -> int {
    INFLLM_TRY(packed_check(c, "packed_evict"));
    if (n < 0 || (n > 0 && !seqs)) return fail(INFLLM_E_BADARG, "packed_evict: %d sequences", n);
    if (budget < 0 || sink < 0 || recent < 0 || sink > budget || recent > budget - sink)
      return fail(INFLLM_E_BADARG, "packed_evict: %lld tokens stay, the first %lld and the newest %lld among them", (long long)budget, (long long)sink, (long long)recent);
    std::vector<infllm_packed_seq> seen(seqs, seqs + n);
    for (auto& s : seen) s.count = s.position = 0;
    INFLLM_TRY(packed_check_seqs(c, seen.data(), n, 0, "packed_evict"));
    int64_t longest = 0;
    for (int i = 0; i < n; ++i) longest = std::max<int64_t>(longest, seqs[i].length);
    if (into) {  // no slot is written to that is read, or written to twice
      for (int i = 0; i < n; ++i) seen.push_back({into[i], 0, 0, 0});
      INFLLM_TRY(packed_check_seqs(c, seen.data(), 2 * n, 0, "packed_evict"));
    }
    if (n == 0 || longest == 0 || (!into && longest <= budget)) return INFLLM_OK;
    const int64_t most_stay = (std::min(budget, longest) + 3) / 4 * 4;
    if (!d_work || (uintptr_t)d_work % 16 || work_bytes < (int64_t)c->n_layers * n * c->n_kv_heads * most_stay * 4)
      return fail(INFLLM_E_BADARG, "packed_evict: a workspace of %lld bytes, 16-byte aligned", (long long)c->n_layers * n * c->n_kv_heads * most_stay * 4);
    DeviceScope scope(c->device);
    EvictParams P;
    P.at = packed_planes(c, 0);
    P.codes_layer = 2 * P.at.codes_v, P.scales_layer = 2 * P.at.scales_v;
    P.weights = c->d_weights, P.places = c->d_places, P.rows_layer = packed_rows(c);
    P.stay = (int32_t*)d_work, P.n_seqs = n, P.most_stay = most_stay;
    P.budget = (int32_t)std::min<int64_t>(budget, INT_MAX), P.sink = (int32_t)std::min(sink, longest), P.recent = (int32_t)std::min(recent, longest);
    P.copy = into != nullptr;
    for (int64_t b0 = 0; b0 < n; b0 += kPackSeqs) {
      const int m = (int)std::min<int64_t>(n - b0, kPackSeqs);
      for (int i = 0; i < m; ++i) P.seq[i] = make_int2(seqs[b0 + i].slot, seqs[b0 + i].length), P.into[i] = into ? into[b0 + i] : 0;
      P.seq0 = b0;
      // as many blocks to a head as the machine has room for
      const int64_t heads = (int64_t)c->n_layers * m * c->n_kv_heads;
      int ctas = 8;
      while (ctas > 1 && heads * ctas > 148 * 4) ctas /= 2;
      P.room = (int32_t)std::min<int64_t>(ceil_div(ceil_div(longest, ctas), kEach) * kEach, kEvictRoom);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)(c->n_kv_heads * ctas), m, c->n_layers);
      cfg.blockDim = dim3(kEvictThreads);
      cfg.dynamicSmemBytes = (size_t)P.room * 4;
      cfg.stream = (cudaStream_t)stream;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim = {(unsigned)ctas, 1, 1};
      cfg.attrs = at, cfg.numAttrs = 1;
      auto kern = c->head_dim == 128 ? packed_evict_kernel<128> : packed_evict_kernel<64>;
      INFLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, P));
      INFLLM_LAUNCH_OK("packed_evict_kernel");
    }
    return INFLLM_OK;
  });
}

// -------------------------------------------------------------------------------------------------------- bookkeeping
namespace {

struct BookSeq {
  int64_t opened, length, position, fresh, change;
};
BookSeq* book_of(infllm_packed_book* b) { return reinterpret_cast<BookSeq*>(b->state); }

int book_check(const infllm_packed_book* b, const int32_t* seqs, int n, const char* what) {
  if (!b || !b->state || b->n_sequences < 1 || b->max_tokens < 1 || n < 0 || (n > 0 && !seqs)) return fail(INFLLM_E_BADARG, "%s: no book, or %d sequences", what, n);
  const BookSeq* s = reinterpret_cast<const BookSeq*>(b->state);
  for (int i = 0; i < n; ++i)
    if (seqs[i] < 0 || seqs[i] >= b->n_sequences || s[seqs[i]].opened % 2 == 0) return fail(INFLLM_E_BADARG, "there is no sequence %d", seqs[i]);
  return INFLLM_OK;
}

}  // namespace

extern "C" int infllm_packed_book_step(infllm_packed_book* book, int what, const int32_t* seqs, const int64_t* opened, int n, const int64_t* counts,
                                       int64_t same, infllm_packed_seq* table, int64_t* as_of, int64_t* info) {
  INFLLM_TRY(book_check(book, seqs, n, "packed_book_step"));
  if (n > 0 && (!opened || (what != INFLLM_PACKED_RETRACT && (!table || !as_of)))) return fail(INFLLM_E_BADARG, "packed_book_step: null pointer");
  if (what < INFLLM_PACKED_EXTEND || what > INFLLM_PACKED_RETRACT || !info) return fail(INFLLM_E_BADARG, "packed_book_step: step %d", what);
  BookSeq* all = book_of(book);
  for (int i = 0; i < n; ++i) {
    const BookSeq& s = all[seqs[i]];
    const int64_t x = counts ? counts[i] : same;
    if (s.opened != opened[i]) return fail(INFLLM_E_BADARG, "sequence %d of this batch has been freed", seqs[i]);
    if (x < 0) return fail(INFLLM_E_BADARG, "%lld tokens", (long long)x);
    if (what == INFLLM_PACKED_EXTEND && x > book->max_tokens - s.length)
      return fail(INFLLM_E_CAPACITY, "sequence %d of %lld tokens and %lld more, where %lld fit", seqs[i], (long long)s.length, (long long)x, (long long)book->max_tokens);
    if (what == INFLLM_PACKED_EXTEND && x > INT32_MAX - s.position) return fail(INFLLM_E_CAPACITY, "sequence %d: a position beyond 31 bits", seqs[i]);
    if (what == INFLLM_PACKED_PLAN && x > s.length) return fail(INFLLM_E_BADARG, "the newest %lld tokens of sequence %d, which has %lld", (long long)x, seqs[i], (long long)s.length);
    if (what == INFLLM_PACKED_RETRACT && x > s.fresh)
      return fail(INFLLM_E_BADARG, "%lld tokens of sequence %d, of which the newest %lld lie in a row", (long long)x, seqs[i], (long long)s.fresh);
  }
  info[0] = info[1] = 0, info[2] = 1;
  for (int i = 0; i < n; ++i) {
    BookSeq& s = all[seqs[i]];
    const int64_t x = counts ? counts[i] : same, more = what == INFLLM_PACKED_EXTEND ? x : what == INFLLM_PACKED_RETRACT ? -x : 0;
    if (what != INFLLM_PACKED_PLAN) s.length += more, s.position += more, s.fresh += more, s.change = ++book->changes;
    if (what == INFLLM_PACKED_RETRACT) continue;
    table[i] = {seqs[i], (int32_t)s.length, (int32_t)x, (int32_t)std::max<int64_t>(s.position - x, 0)};
    as_of[i] = s.change;
    info[0] = std::max(info[0], x);
    if (x > 0) info[1] = std::max(info[1], s.position);
    if (x > s.fresh) info[2] = 0;
  }
  return INFLLM_OK;
}

extern "C" int infllm_packed_book_evict(infllm_packed_book* book, const int32_t* seqs, int n, const int32_t* into, int64_t budget, int64_t sink,
                                        int64_t recent, infllm_packed_seq* table, int64_t* most, int apply) {
  return guarded("packed_book_evict", [&]() -> int {
    INFLLM_TRY(book_check(book, seqs, n, "packed_book_evict"));
    if (into) INFLLM_TRY(book_check(book, into, n, "packed_book_evict"));
    BookSeq* all = book_of(book);
    if (!apply) {
      if (!most || (n > 0 && !table)) return fail(INFLLM_E_BADARG, "packed_book_evict: null pointer");
      if (budget < 0 || sink < 0 || recent < 0 || sink > budget || recent > budget - sink)
        return fail(INFLLM_E_BADARG, "%lld tokens stay, the first %lld and the newest %lld among them", (long long)budget, (long long)sink, (long long)recent);
      std::vector<int32_t> names(seqs, seqs + n);
      if (into) names.insert(names.end(), into, into + n);
      std::sort(names.begin(), names.end());
      for (size_t i = 1; i < names.size(); ++i)
        if (names[i] == names[i - 1]) return fail(INFLLM_E_BADARG, "sequence %d twice", names[i]);
      *most = 0;
      for (int i = 0; i < n; ++i) {
        const int64_t length = all[seqs[i]].length;
        table[i] = {seqs[i], (int32_t)length, 0, 0};
        *most = std::max(*most, std::min(length, budget));
      }
      return INFLLM_OK;
    }
    for (int i = 0; i < n; ++i) {
      const BookSeq s = all[seqs[i]];
      if (!into && s.length <= budget) continue;
      BookSeq& to = all[into ? into[i] : seqs[i]];
      to.length = std::min(s.length, budget), to.position = s.position;
      to.fresh = s.length <= budget ? s.fresh : std::min(s.fresh, recent);
      to.change = ++book->changes;
    }
    return INFLLM_OK;
  });
}
