// Attention of a batch of sequences over the cache in 4 bits (packed.cuh), and the weights that it gives the cache's tokens.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij) / sum_j exp(s_ij),  s_ij = scale q_i . k_j,  over the keys j up to query i's place
//   w_j = decay w_j + sum_i p_ij, over the counted queries of all query heads of a KV head
//
// Keys are cut into stretches, the parts of a row joined by their log-sum-exps,
//   M = max_p lse_p,   o = sum_p 2^(lse_p - M) o_p / sum_p 2^(lse_p - M)   (logarithms to base 2).
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>

#include "attn_tc.cuh"
#include "decode_warp.cuh"
#include "packed_attn.cuh"

namespace infllm {

using namespace mma;

constexpr int kAttnWarps = 4, kFewRows = 8;

// loads of 16, 8 and 4 bytes that are read once, kAt bytes behind an address
template <int kAt>
__device__ __forceinline__ uint4 ld_stream16(const char* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4+%5];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p), "n"(kAt));
  return r;
}
template <int kAt>
__device__ __forceinline__ uint2 ld_stream8(const char* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2+%3];" : "=r"(r.x), "=r"(r.y) : "l"(p), "n"(kAt));
  return r;
}
template <int kAt>
__device__ __forceinline__ uint32_t ld_stream4(const char* p) {
  uint32_t r;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1+%2];" : "=r"(r) : "l"(p), "n"(kAt));
  return r;
}

// ------------------------------------------------------------------------------------------------------- few rows
// Up to eight rows of a KV head.  A warp takes groups of 16 keys, keys and values from global memory through registers into operands of the
// m16n8k16 products:
//   S^T = K Q^T       keys are rows: a thread's codes of a key are the numbers of one (m, s) (kDim 128) or of half a one
//   O^T += V^T P^T    numbers of the values are rows: a thread's codes of a value are an eighth of it, and two keys' are paired as they
//                     are taken out.  P^T is S^T's place with keys and rows exchanged: two 8 x 8 transpositions in the warp.
// P is two 16-bit numbers, p = hi + lo, so that an output's only rounding is its own: where rows are no more than four (kFour), the other
// four columns have the same rows again, and theirs is lo, in the same product.  In fp16, whose numbers end at 2^-24, lo is kept times
// 2^11, as it is that much smaller than hi wherever hi has all its digits: the other four columns are scaled at the end; with more rows the
// products of lo are formed apart and added, a multiplication and addition of O's numbers for 16 keys.  (Without the two an fp16 call of 32
// sequences takes 215 us instead of 217, below; of eight rows, 16 sequences with 64/8 heads, 134 instead of 139.)
// The reference of a row is lazy (packed_attn.cuh): only where it moves O is scaled and do lanes exchange anything.
// What bounds it: the codes' bytes, and close behind them what is issued to take numbers out of them, 397 instructions a warp for 16 keys of
// 128 (loads alone 138 us where the kernel took 192; without the taking out 189).  One new token of 32 sequences of 24576 tokens, 32/8
// heads of 128 in bf16: 1.007 GB in 190 us, 5.30 TB/s (fp16 216); of 16, 64/8 heads, 111 (126); of one sequence of 131072, 168 MB in 39 us.
// What brought it there from 389: loads of the next 16 keys under this one's products, two copies of a turn so that their registers stay where they are, Q in shared memory (four
// blocks a multiprocessor by registers), keys as rows of S^T so that a thread's codes have one (m, s), and addresses that run.  Tried, and
// slower: 32 keys at a time (the kernel of then 291 instead of 286), five blocks a multiprocessor (324), lines asked for into L2 ahead
// (275, 265), shifts and differences instead of the masks of packed.cuh (a tenth more).
template <typename T, int kDim, bool kFour>
struct PackedRows {
  static constexpr int kW = kDim / 32;  // words of a key, kDim / 4 numbers, that a thread has: as many of Q's 16-byte pieces
  static constexpr int kH = kDim / 64;  // of a value, kDim / 8 numbers
  static constexpr int kRow = kDim / 2, kScales = kDim / 8, kTiles = 4 * kH;
  static constexpr float kGrow = Reference<T>::kGrow, kBelow = Reference<T>::kBelow;
  static constexpr bool kApart = !Reference<T>::kBf16;  // lo is kept times 2^11
  static constexpr float kLo = kApart ? 2048.f : 1.f, kUnLo = 1.f / kLo;
  // the reference before there is one: any score that fits 32 bits is above it, and what a row does not see, or does not fit, -inf, is a
  // probability of 0 beside it
  static constexpr float kNone = -FLT_MAX;
  using C = Codes<T>;
  const uint4* qf;     // row g's pieces, in shared memory: [piece][lane].  (The registers are worth more than four loads a group.)
  int lim[2];          // keys that rows 2t and 2t + 1 see
  float ot[kTiles][4];  // O^T: [0], [1] = number g * kDim / 8 + 2i of columns 2t, 2t + 1; [2], [3] = the next one
  float m[2], l[2];

  struct Key {  // rows nt * 8 + g
    uint32_t w[2][kW], ms[2];
    // codes and scales from here on: this thread's of row nt
    template <int kNt>
    __device__ __forceinline__ void load(const char* codes, const char* scales) {
      if constexpr (kDim == 128) {
        const uint4 x = ld_stream16<kNt * 8 * kRow>(codes);
        w[kNt][0] = x.x, w[kNt][1] = x.y, w[kNt][2] = x.z, w[kNt][3] = x.w;
      } else {
        const uint2 x = ld_stream8<kNt * 8 * kRow>(codes);
        w[kNt][0] = x.x, w[kNt][1] = x.y;
      }
      ms[kNt] = ld_stream4<kNt * 8 * kScales>(scales);
    }
  };
  struct Value {  // rows 2t, 2t + 1, 2t + 8, 2t + 9
    uint32_t w[4][kH], ms[4];
    template <int kKi>
    __device__ __forceinline__ void load(const char* codes, const char* scales) {
      constexpr int kR = (kKi & 1) + (kKi >> 1) * 8;
      if constexpr (kDim == 128) {
        const uint2 x = ld_stream8<kR * kRow>(codes);
        w[kKi][0] = x.x, w[kKi][1] = x.y;
      } else {
        w[kKi][0] = ld_stream4<kR * kRow>(codes);
      }
      ms[kKi] = ld_stream4<kR * kScales>(scales);
    }
  };
  // where a thread's pieces of 16 keys begin, from the first one's codes and scales of keys and of values on
  struct Place {
    const char *kc, *ks, *vc, *vs;
    __device__ __forceinline__ Place(const char* codes, const char* scales, int64_t codes_v, int64_t scales_v) {
      const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
      kc = codes + g * kRow + t * (kRow / 4), ks = scales + g * kScales + (kDim == 128 ? t : t >> 1) * 4;
      vc = codes + codes_v + 2 * t * kRow + g * (kRow / 8), vs = scales + scales_v + 2 * t * kScales + (kDim == 128 ? g >> 1 : g >> 2) * 4;
    }
    __device__ __forceinline__ void advance(int keys) { kc += keys * kRow, ks += keys * kScales, vc += keys * kRow, vs += keys * kScales; }
    __device__ __forceinline__ void load(Key& k, Value& v) const {
      k.template load<0>(kc, ks);
      k.template load<1>(kc, ks);
      v.template load<0>(vc, vs);
      v.template load<1>(vc, vs);
      v.template load<2>(vc, vs);
      v.template load<3>(vc, vs);
    }
    // nk keys are there: what lies behind the last is not read, as it may not be a number, and 0 times that is none
    __device__ __forceinline__ void load(Key& k, Value& v, int nk) const {
      const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int64_t back = min(nk - 1 - (nt * 8 + g), 0);  // rows from the one that would be this thread's
        Key x;
        if (nt == 0) x.template load<0>(kc + back * kRow, ks + back * kScales);
        else x.template load<1>(kc + back * kRow, ks + back * kScales);
#pragma unroll
        for (int j = 0; j < kW; ++j) k.w[nt][j] = x.w[nt][j];
        k.ms[nt] = x.ms[nt];
      }
#pragma unroll
      for (int ki = 0; ki < 4; ++ki) {
        const int64_t back = min(nk - 1 - (2 * t + (ki & 1) + (ki >> 1) * 8), 0);
        Value x;
        if (ki == 0) x.template load<0>(vc + back * kRow, vs + back * kScales);
        else if (ki == 1) x.template load<1>(vc + back * kRow, vs + back * kScales);
        else if (ki == 2) x.template load<2>(vc + back * kRow, vs + back * kScales);
        else x.template load<3>(vc + back * kRow, vs + back * kScales);
#pragma unroll
        for (int j = 0; j < kH; ++j) v.w[ki][j] = x.w[ki][j];
        v.ms[ki] = x.ms[ki];
      }
    }
  };

  __device__ __forceinline__ void clear() {
    m[0] = m[1] = kNone, l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) ot[i][0] = ot[i][1] = ot[i][2] = ot[i][3] = 0.f;
  }
  static __device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  static __device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
  }

  // 16 keys from j0 on; kAll: every row sees all of them.  Otherwise those below key1, and a row those below its own limit.
  // kWeigh: scores are left for the weights; logits: the place of this thread's first row's of key g, null: it has none
  template <bool kAll, bool kWeigh>
  __device__ __forceinline__ void group(const Key& k, const Value& v, int j0, int key1, float scale_log2, float* logits, int64_t pitch, bool two) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float s[4] = {0.f, 0.f, 0.f, 0.f};  // key g of rows 2t, 2t + 1; key g + 8
    {
      const auto m0 = C::least2(k.ms[0]), s0 = C::step2(k.ms[0]), m1 = C::least2(k.ms[1]), s1 = C::step2(k.ms[1]);
#pragma unroll
      for (int j = 0; j < kW; ++j) {
        const uint4 q = qf[j * 32];
        uint32_t a[4], b[4];
        C::pairs(k.w[0][j], m0, s0, a);
        C::pairs(k.w[1][j], m1, s1, b);
        const uint32_t x[4] = {a[0], b[0], a[1], b[1]}, y[4] = {a[2], b[2], a[3], b[3]};
        mma16816<T>(s, x, q.x, q.y);
        mma16816<T>(s, y, q.z, q.w);
      }
    }
    if (!kAll) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j0 + (e >> 1) * 8 + g >= min(lim[e & 1], key1)) s[e] = -INFINITY;
    }
    if (kWeigh && logits) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((kAll || j0 + (e >> 1) * 8 + g < key1) && (!(e & 1) || two)) logits[(e & 1) * pitch + j0 + (e >> 1) * 8] = s[e] * scale_log2;
    }
    float mx[2] = {fmaxf(s[0], s[2]) * scale_log2, fmaxf(s[1], s[3]) * scale_log2};
    if (__any_sync(0xffffffffu, mx[0] > m[0] + kGrow || mx[1] > m[1] + kGrow)) {
      float al[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], o));
        const float mn = mx[e] > m[e] + kGrow ? mx[e] - kBelow : m[e];
        al[e] = exp2f(m[e] - mn);
        m[e] = mn;
        l[e] *= al[e];
      }
#pragma unroll
      for (int i = 0; i < kTiles; ++i) ot[i][0] *= al[0], ot[i][1] *= al[1], ot[i][2] *= al[0], ot[i][3] *= al[1];
    }
    const float p[4] = {ex2(fmaf(s[0], scale_log2, -m[0])), ex2(fmaf(s[1], scale_log2, -m[1])), ex2(fmaf(s[2], scale_log2, -m[0])), ex2(fmaf(s[3], scale_log2, -m[1]))};
    l[0] += p[0] + p[2];
    l[1] += p[1] + p[3];
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      typename Act<T>::T2 h = Act<T>::from_f2(p[2 * e], p[2 * e + 1]);
      hi[e] = *reinterpret_cast<uint32_t*>(&h);
      const float2 f = Act<T>::to_f2(h);
      lo[e] = pack2<T>((p[2 * e] - f.x) * kLo, (p[2 * e + 1] - f.y) * kLo);
      if (kFour) hi[e] = t < 2 ? hi[e] : lo[e];
      hi[e] = transposed(hi[e]);
      if (!kFour) lo[e] = transposed(lo[e]);
    }
    // A operands: numbers of keys 2t, 2t + 1 and of 2t + 8, 2t + 9
    const auto m01 = C::least2(v.ms[0], v.ms[1]), s01 = C::step2(v.ms[0], v.ms[1]);
    const auto m23 = C::least2(v.ms[2], v.ms[3]), s23 = C::step2(v.ms[2], v.ms[3]);
#pragma unroll
    for (int j = 0; j < kH; ++j) {
      uint32_t e01[4], o01[4], e23[4], o23[4];
      C::pairs(__byte_perm(v.w[0][j], v.w[1][j], 0x5410), m01, s01, e01);
      C::pairs(__byte_perm(v.w[0][j], v.w[1][j], 0x7632), m01, s01, o01);
      C::pairs(__byte_perm(v.w[2][j], v.w[3][j], 0x5410), m23, s23, e23);
      C::pairs(__byte_perm(v.w[2][j], v.w[3][j], 0x7632), m23, s23, o23);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a[4] = {e01[i], o01[i], e23[i], o23[i]};
        mma16816<T>(ot[j * 4 + i], a, hi[0], hi[1]);
        if (!kFour && !kApart) mma16816<T>(ot[j * 4 + i], a, lo[0], lo[1]);
        if (!kFour && kApart) {
          float z[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816<T>(z, a, lo[0], lo[1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) ot[j * 4 + i][e] = fmaf(z[e], kUnLo, ot[j * 4 + i][e]);
        }
      }
    }
  }
};

// Four warps share a stretch's groups of 16 keys and meet in shared memory.
template <typename T, int kDim, bool kFour, bool kWeigh>
__global__ void __launch_bounds__(kAttnWarps * 32, 4) packed_rows_kernel(const __grid_constant__ PackedAttnParams P) {
  using R = PackedRows<T, kDim, kFour>;
  using C = Codes<T>;
  constexpr int kPitch = kDim + 4, kStep = kAttnWarps * 16;
  __shared__ __align__(16) float sm_o[kAttnWarps][8][kPitch];
  __shared__ float sm_m[kAttnWarps][8], sm_l[kAttnWarps][8];
  __shared__ uint4 sm_q[R::kW][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int unit = blockIdx.x, hkv = blockIdx.y, b = seq_of(P, unit);
  const PackedAttnSeq S = P.seq[b];
  const int key0 = (unit - S.unit0) * S.keys, rows = S.count * P.group;
  const int key1 = min(key0 + S.keys, S.length);
  const int least = keys_of_row(S, P.group, 0);  // keys that every row sees
  R w;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = kFour ? (2 * t + e) & 3 : 2 * t + e;
    w.lim[e] = r < rows ? keys_of_row(S, P.group, r) : 0;
  }
  const int64_t first = P.at.row0(S.slot, hkv) + key0 + warp * 16;  // of the stretch, this warp's first row
  typename R::Place at(P.at.codes + first * R::kRow, P.at.scales + first * R::kScales, P.at.codes_v, P.at.scales_v);
  float* logits = nullptr;
  if (kWeigh && 2 * t < rows) logits = P.logits + (((int64_t)(P.b0 + b) * P.at.n_kv + hkv) * P.logit_rows + 2 * t) * P.pitch + g;
  const bool two = 2 * t + 1 < rows;
  chain_enter();
  if (warp < R::kW) {  // a piece of every row by a warp
    const int r = kFour ? g & 3 : g, i = r / P.group, h = r - i * P.group;
    const char* from = P.q + (int64_t)(P.b0 + b) * P.q_bs + (int64_t)(hkv * P.group + h) * P.q_hs + (int64_t)(P.most - S.count + i) * P.q_ts;
    sm_q[warp][lane] = r < rows ? __ldg(reinterpret_cast<const uint4*>(from + t * (kDim / 2) + warp * 16)) : make_uint4(0, 0, 0, 0);
  }
  w.qf = &sm_q[0][lane];
  w.clear();
  const int whole = min(key1, least) - 16;  // the last place of a group that all rows see all of
  int j0 = key0 + warp * 16;
  // A group is on its way while the one before it is worked on: two copies of the work, each with its own registers, as what is on its
  // way is not to be moved, which would wait for it.
  typename R::Key k0, k1;
  typename R::Value v0, v1;
  if (j0 <= whole) at.load(k0, v0);
  __syncthreads();
  if (j0 <= whole) {
    auto turn = [&](const typename R::Key& k, const typename R::Value& v, typename R::Key& kn, typename R::Value& vn) {
      const bool more = j0 + kStep <= whole;
      at.advance(kStep);
      if (more) at.load(kn, vn);
      w.template group<true, kWeigh>(k, v, j0, key1, P.scale_log2, logits, P.pitch, two);
      j0 += kStep;
      return more;
    };
    while (turn(k0, v0, k1, v1) && turn(k1, v1, k0, v0)) {
    }
  }
  // Keys that some rows do not see: a value that is no number must not reach those, and 0 times it is none.  Its group is 0 here, and from its
  // place on the rows that see it become none in the end, in these numbers alone.
  int none = INT_MAX;  // the first such key, of the group that this thread's numbers are of
#pragma unroll 1
  for (; j0 < key1; j0 += kStep, at.advance(kStep)) {
    typename R::Key k;
    typename R::Value v;
    const int nk = min(16, key1 - j0);
    at.load(k, v, nk);
#pragma unroll
    for (int ki = 0; ki < 4; ++ki)
      if (C::odd(v.ms[ki])) v.ms[ki] = 0, none = min(none, j0 + min(2 * t + (ki & 1) + (ki >> 1) * 8, nk - 1));
    w.template group<false, kWeigh>(k, v, j0, key1, P.scale_log2, logits, P.pitch, two);
  }
  none = min(none, __shfl_xor_sync(0xffffffffu, none, 1));
  none = min(none, __shfl_xor_sync(0xffffffffu, none, 2));
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) w.l[e] += __shfl_xor_sync(0xffffffffu, w.l[e], o);
    if (w.m[e] == R::kNone) w.m[e] = w.l[e] != w.l[e] ? 0.f : -INFINITY;  // (scores that are no numbers are not seen by the maximum)
    if (g == 0) sm_m[warp][2 * t + e] = w.m[e], sm_l[warp][2 * t + e] = w.l[e];
    if (none < w.lim[e]) {
#pragma unroll
      for (int i = 0; i < R::kTiles; ++i) w.ot[i][e] = w.ot[i][2 + e] = NAN;
    }
#pragma unroll
    for (int i = 0; i < R::kTiles; ++i) *reinterpret_cast<float2*>(&sm_o[warp][2 * t + e][g * (kDim / 8) + 2 * i]) = make_float2(w.ot[i][e], w.ot[i][2 + e]);
  }
  __syncthreads();
  for (int idx = tid; idx < rows * (kDim / 2); idx += kAttnWarps * 32) {  // two neighbouring numbers each
    const int r = idx / (kDim / 2), d = idx % (kDim / 2) * 2;
    float mx = sm_m[0][r];
#pragma unroll
    for (int y = 1; y < kAttnWarps; ++y) mx = fmaxf(mx, sm_m[y][r]);
    float den = 0.f, n0 = 0.f, n1 = 0.f;
    if (mx != -INFINITY) {
#pragma unroll
      for (int y = 0; y < kAttnWarps; ++y) {
        const float wt = exp2f(sm_m[y][r] - mx);
        den = fmaf(wt, sm_l[y][r], den);
        n0 = fmaf(wt, kFour ? fmaf(sm_o[y][r + 4][d], R::kUnLo, sm_o[y][r][d]) : sm_o[y][r][d], n0);
        n1 = fmaf(wt, kFour ? fmaf(sm_o[y][r + 4][d + 1], R::kUnLo, sm_o[y][r][d + 1]) : sm_o[y][r][d + 1], n1);
      }
      n0 /= den, n1 /= den;
    }
    const float lse = mx == -INFINITY ? -INFINITY : mx + log2f(den);
    const int64_t pr = ((int64_t)unit * P.at.n_kv + hkv) * kFewRows + r;
    if (d == 0 && (S.chunks > 1 || kWeigh)) P.part_lse[pr] = lse;
    if (S.chunks > 1) {
      *reinterpret_cast<float2*>(P.part_o + pr * kDim + d) = make_float2(n0, n1);
    } else {
      const int i = r / P.group, h = r - i * P.group;
      const int64_t orow = ((int64_t)(P.b0 + b) * P.most + P.most - S.count + i) * (P.at.n_kv * P.group) + hkv * P.group + h;
      *reinterpret_cast<uint32_t*>(P.out + (orow * kDim + d) * 2) = pack2<T>(n0, n1);
      if (P.lse && d == 0) P.lse[orow] = lse * (1.f / kLog2e);
    }
  }
}

// ----------------------------------------------------------------------------------------------------------- the join
// The weights of four keys a thread from the scores that the kernel of few rows has left, 1024 keys of a KV head a block.
constexpr int kSumKeys = 1024;
__device__ __forceinline__ void sum_weights(const PackedAttnParams& P, int block) {
  __shared__ float sm_lse[8];
  const int per = (int)(P.pitch / kSumKeys), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hkv = block / per % P.at.n_kv, b = block / per / P.at.n_kv;
  const PackedAttnSeq S = P.seq[b];
  const int key0 = block % per * kSumKeys, rows = S.count * P.group, from = (S.count - min(P.weigh, S.count)) * P.group;
  chain_enter();
  if (rows == 0 || key0 >= S.length) return;
  if (warp < rows) {  // a row's log-sum-exp, of its parts'
    float mx = -INFINITY, sum = 0.f;
    auto part = [&](int c) { return P.part_lse[((int64_t)(S.unit0 + c) * P.at.n_kv + hkv) * kFewRows + warp]; };
    for (int c = lane; c < S.chunks; c += 32) mx = fmaxf(mx, part(c));
    mx = warp_max(mx);
    if (mx == -INFINITY) mx = 0.f;  // (where all are no numbers)
    for (int c = lane; c < S.chunks; c += 32) sum += exp2f(part(c) - mx);
    sum = warp_sum(sum);
    if (lane == 0) sm_lse[warp] = mx + log2f(sum);
  }
  __syncthreads();
  const int key = key0 + threadIdx.x * 4;
  if (key >= S.length) return;
  const float* from_logits = P.logits + ((int64_t)(P.b0 + b) * P.at.n_kv + hkv) * P.logit_rows * P.pitch + key;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r = from; r < rows; ++r) {
    const float4 s = *reinterpret_cast<const float4*>(from_logits + r * P.pitch);
    const float z = sm_lse[r];
    w[0] += exp2f(s.x - z), w[1] += exp2f(s.y - z), w[2] += exp2f(s.z - z), w[3] += exp2f(s.w - z);
  }
  float* to = P.weights + P.at.row0(S.slot, hkv) + key;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (key + e < S.length) to[e] = P.decay == 0.f ? w[e] : P.decay * to[e] + w[e];
  }
}

// A row's parts, by kWarps warps that share them, four on their way at once: sum, maximum and kDim / 32 numbers a lane, in the first
// of the warps (false in the others).  row_of(part): its row in part_lse and part_o.
template <int kDim, int kWarps, bool kTc, typename F>
__device__ __forceinline__ bool join_row(const PackedAttnParams& P, int parts, F&& row_of, float& m, float& l, float (&acc)[kDim / 32]) {
  constexpr int kPer = kDim / 32, kAhead = 4;
  __shared__ float sm[8][kDim + 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
  for (int c0 = warp % kWarps; c0 < parts; c0 += kWarps * kAhead) {
    float lse[kAhead], v[kAhead][kPer];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int c = c0 + e * kWarps;
      lse[e] = -INFINITY;
      if (c >= parts) continue;
      const int64_t row = row_of(c);
      lse[e] = P.part_lse[row];
      // (partial rows of the tensor-core kernel lie in blocks of 32, four columns of all of them side by side)
      const float* o = P.part_o + (kTc ? (row & ~(int64_t)31) * kDim + (lane * kPer / 4) * 128 + (row & 31) * 4 + lane * kPer % 4 : row * kDim + lane * kPer);
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
  if (kWarps > 1) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) sm[warp][lane * kPer + k] = acc[k];
    if (lane == 0) sm[warp][kDim] = m, sm[warp][kDim + 1] = l;
    __syncthreads();
    if (warp % kWarps) return false;
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
  return true;
}

// a joined row: token i (of the tensors) of query head h of the launch's sequence b; its log-sum-exp to base 2
template <typename T, int kDim>
__device__ __forceinline__ float write_row(const PackedAttnParams& P, int b, int i, int h, float m, float l, const float (&acc)[kDim / 32]) {
  constexpr int kPer = kDim / 32;
  const int lane = threadIdx.x & 31;
  const int64_t orow = ((int64_t)(P.b0 + b) * P.most + i) * (P.at.n_kv * P.group) + h;
  const float inv = l > 0.f ? 1.f / l : l;  // (a NaN stays one)
  uint32_t* to = reinterpret_cast<uint32_t*>(P.out + (orow * kDim + lane * kPer) * 2);
#pragma unroll
  for (int k = 0; k < kPer; k += 2) to[k / 2] = pack2<T>(acc[k] * inv, acc[k + 1] * inv);
  const float lse = l > 0.f ? m + log2f(l) : l == 0.f ? -INFINITY : l;
  if (lane == 0 && P.lse) P.lse[orow] = lse * (1.f / kLog2e);
  return lse;
}

// few rows: all of a launch's rows, those without a token as zeros
template <typename T, int kDim, int kWarps>
__global__ void __launch_bounds__(256) packed_join_kernel(const __grid_constant__ PackedAttnParams P) {
  if ((int)blockIdx.x >= P.join_blocks) {
    sum_weights(P, blockIdx.x - P.join_blocks);
    return;
  }
  const int warp = threadIdx.x >> 5, heads = P.at.n_kv * P.group;
  const int64_t at = (int64_t)blockIdx.x * (8 / kWarps) + warp / kWarps;
  const bool in = at < (int64_t)P.batch * P.most * heads;
  const int h = in ? (int)(at % heads) : 0, i = in ? (int)(at / heads % P.most) : 0, b = in ? (int)(at / heads / P.most) : 0, hkv = h / P.group;
  const PackedAttnSeq S = P.seq[b];
  const int tok = i - (P.most - S.count), r = tok * P.group + h % P.group;
  const bool whole = tok >= 0 && S.chunks == 1;  // written by the unit that had all of it
  chain_enter();
  float m, l, acc[kDim / 32];
  const bool mine = join_row<kDim, kWarps, false>(P, in && tok >= 0 && !whole ? S.chunks : 0, [&](int c) -> int64_t { return ((int64_t)(S.unit0 + c) * P.at.n_kv + hkv) * kFewRows + r; }, m, l, acc);
  if (mine && in && !whole) write_row<T, kDim>(P, b, i, h, m, l, acc);
}

// many rows: those of the units that were cut, a block of the grid's second dimension for each block in which a unit begins that ends in another one
template <typename T, int kDim, int kWarps>
__global__ void __launch_bounds__(256) packed_join_cut_kernel(const __grid_constant__ PackedTcParams All) {
  const PackedAttnParams& P = All.a;
  const int first = blockIdx.y, warp = threadIdx.x >> 5;
  const int2 begin = All.start[first], end = All.start[first + 1];
  chain_enter();
  // the unit that the block's stretch ends in, if the stretch has its first tile and not its last
  if (end.y == 0 || (begin.x == end.x && begin.y > 0)) return;
  const int unit = end.x, b = seq_of(P, unit);
  const PackedAttnSeq S = P.seq[b];
  const int hkv = (unit - S.unit0) / S.chunks, block = (unit - S.unit0) % S.chunks, in_block = blockIdx.x * (8 / kWarps) + warp / kWarps;
  const int r = block * kBlockRows + in_block, parts = block_of(All, unit, tiles_of(S, P.group, block) - 1) - first + 1;
  const bool in = r < S.count * P.group;
  // a block's first unit has its first slot, its last one the second
  float m, l, acc[kDim / 32];
  const bool mine = join_row<kDim, kWarps, true>(P, in ? parts : 0, [&](int c) -> int64_t { return (int64_t)(2 * (first + c) + (All.start[first + c].x < unit)) * kBlockRows + in_block; }, m, l, acc);
  if (!mine || !in) return;
  const int tok = r / P.group;
  const float lse = write_row<T, kDim>(P, b, P.most - S.count + tok, hkv * P.group + r - tok * P.group, m, l, acc);
  if ((threadIdx.x & 31) == 0 && P.row_lse) P.row_lse[((int64_t)(P.b0 + b) * P.at.n_kv + hkv) * P.most * P.group + r] = lse;
}

// rows of tokens that are none, where sequences have fewer than the tensors: a warp a row
template <typename T, int kDim>
__global__ void __launch_bounds__(256) packed_empty_kernel(const __grid_constant__ PackedAttnParams P) {
  const int heads = P.at.n_kv * P.group, b = blockIdx.y;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  chain_enter();
  if (at >= (int64_t)(P.most - P.seq[b].count) * heads) return;
  const float none[kDim / 32] = {};
  write_row<T, kDim>(P, b, (int)(at / heads), (int)(at % heads), -INFINITY, 0.f, none);
}

// as many warps to a row as one wave has room for
template <typename F>
static int by_warps(int64_t rows, int n_sm, F&& launch) {
  const int64_t warps = n_sm * 32 / std::max<int64_t>(rows, 1);
  INFLLM_CUDA_OK(warps >= 8 ? launch(std::integral_constant<int, 8>()) : warps >= 2 ? launch(std::integral_constant<int, 2>()) : launch(std::integral_constant<int, 1>()));
  INFLLM_LAUNCH_OK("packed_join_kernel");
  return INFLLM_OK;
}

namespace {

// Keys of a unit's stretch.  A multiprocessor takes kGroup microseconds to a block's 64 keys while it has blocks to spare, kTwo to two blocks'
// and kAlone to one's; a wave of blocks costs kWave besides, and a join kJoin.  (Fitted to ten batches of 1 to 64 sequences, each with
// stretches of 64 to 6144 keys; what is chosen takes up to 8 % more than the best of those.)
int64_t chunk_keys(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int n_sm) {
  constexpr double kGroup = .3, kTwo = .7, kAlone = .42, kWave = 2.5, kJoin = 4.;
  int64_t most = 64, groups = 0;  // (up to 2^24 keys, so that a stretch's bytes are counted in 32 bits)
  for (int i = 0; i < n; ++i) {
    if (seqs[i].count == 0) continue;
    most = std::max<int64_t>(most, std::min<int64_t>(ceil_div(seqs[i].length, 64) * 64, 1 << 24));
    groups += ceil_div(seqs[i].length, 64);
  }
  auto units = [&](int64_t keys) {
    int64_t u = 0;
    for (int i = 0; i < n; ++i) u += seqs[i].count > 0 ? (uint32_t)(seqs[i].length + keys - 1) / (uint32_t)keys : 0;
    return u * c->n_kv_heads;
  };
  int64_t best = most, tried = 0;
  double least = 1e300;
  for (int each = 1; each <= 32; each += each < 14 ? 1 : 6) {  // blocks of a multiprocessor
    const int64_t room = (int64_t)each * n_sm;
    int64_t keys = std::min(most, std::max<int64_t>(1, groups * c->n_kv_heads / room) * 64), u = units(keys);
    while (u > room && keys < most) keys = std::min(most, std::max(keys + 64, keys * std::min(u, 2 * room) / room / 64 * 64)), u = units(keys);
    for (int down = 0; down < 8 && keys > 64 && units(keys - 64) == u; ++down) keys -= 64;
    if (keys == tried) continue;
    tried = keys;
    const int64_t per = ceil_div(u, n_sm);
    // (equal blocks run in waves; where lengths differ, short ones fill up what the long ones leave, but for the last)
    const double each_full = (double)(keys / 64) * (per > 2 ? kGroup * (double)per : per == 2 ? kTwo : kAlone);
    const double filled = kGroup * (double)(groups * c->n_kv_heads) / n_sm + kAlone * (double)(keys / 64);
    const double cost = std::min(each_full, filled) + kWave * (double)ceil_div(per, 4) + (keys < most ? kJoin : 0.);
    if (cost < least) least = cost, best = keys;
    if (keys == 64) break;
  }
  return best;
}

// multiprocessors of a device (of a B200 where there is none: sizes are worked out without one, too)
int sm_count(int device) {
  static std::atomic<int> known[64];
  if (device < 0 || device >= 64) return 148;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
      cudaGetLastError();
      return 148;
    }
    n = std::min(n, kMaxSms);
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Work, in half microseconds
constexpr int64_t kUnitWork = 8;   // of a unit of many rows besides its tiles
constexpr int64_t kBlockWork = 24;  // worth a block
int64_t tile_work(int64_t rows) { return rows > 128 ? 4 : 2; }  // of 128 keys

// whether a call goes to the kernel of many rows: some sequence has more than eight
bool many_rows(const infllm_packed_seq* seqs, int n, int group) {
  int64_t most = 0;
  for (int i = 0; i < n; ++i) most = std::max<int64_t>(most, (int64_t)seqs[i].count * group);
  return most > kFewRows;
}
// keys that a row of scores has room for
int64_t logit_pitch(const infllm_packed_seq* seqs, int n) {
  int64_t longest = 0;
  for (int i = 0; i < n; ++i) longest = std::max<int64_t>(longest, seqs[i].length);
  return ceil_div(longest, kSumKeys) * kSumKeys;
}

// the units of the launch of seqs[0 .. n - 1] for few rows: stretches of a sequence's keys
int64_t lay_out_few(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int n_sm, PackedAttnSeq* to, bool* join) {
  const int64_t keys = chunk_keys(c, seqs, n, n_sm);
  int64_t u = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t chunks = seqs[i].count > 0 ? ceil_div(seqs[i].length, keys) : 0;
    to[i] = {seqs[i].slot, seqs[i].length, seqs[i].count, (int32_t)std::min<int64_t>(u, INT_MAX), (int32_t)chunks, (int32_t)keys};
    *join = *join || chunks > 1;
    u += chunks;
  }
  return u;
}

// Deals the tiles of units 0, 1, .. out to blocks, so that all have about the same work: for_each calls f(tiles, work of one).
template <typename F>
void deal_out(PackedTcParams& P, int n_sm, bool* join, F&& for_each) {
  int64_t work = 0;
  for_each([&](int64_t tiles, int64_t each) { work += kUnitWork + tiles * each; });
  // (a cut costs a unit's start; where that was too little, so that the last block has more than the others, shares grow)
  int64_t share = std::max(ceil_div(work, n_sm) + kUnitWork, kBlockWork), left = 0;
  int ctas = 0, u = 0;
  bool cut = false;
  for (int tries = 0; tries < 20; ++tries, share += ceil_div(share, 16)) {
    ctas = u = 0, left = 0, cut = false;
    for_each([&](int64_t tiles, int64_t each) {
      int64_t at = 0;
      while (at < tiles) {
        // short ends stay where they are
        if (ctas == 0 || (left < kUnitWork + 4 * each && left < kUnitWork + (tiles - at) * each && ctas < n_sm))
          P.start[ctas++] = make_int2(u, (int)at), left = share;
        int64_t take = tiles - at;
        if (ctas < n_sm && kUnitWork + take * each > left + 2 * each) take = std::max<int64_t>(1, std::min(take, (left - kUnitWork) / each));
        left -= kUnitWork + take * each;
        cut = cut || take < tiles;
        at += take;
      }
      ++u;
    });
    if (left > -share / 16 - 8) break;
  }
  P.start[ctas] = make_int2(u, 0);
  P.n_ctas = ctas;
  *join = *join || cut;
}

int many_units(const infllm_packed* c, const infllm_packed_seq* seqs, PackedTcParams& P, int kv_units(const infllm_packed_seq&, int)) {
  int64_t u = 0;
  for (int i = 0; i < P.a.batch; ++i) {
    const int blocks = kv_units(seqs[i], P.a.group);
    P.a.seq[i] = {seqs[i].slot, seqs[i].length, seqs[i].count, (int32_t)u, std::max(blocks, 1), 0};
    u += (int64_t)blocks * c->n_kv_heads;
    if (u > INT_MAX) return fail(INFLLM_E_BADARG, "packed_attend: %lld units of work", (long long)u);
  }
  return INFLLM_OK;
}

// Bytes of the image of a launch's tiles, and of a word for each, 0 where numbers are taken out of their codes by the blocks themselves: with an image a tile of 256
// rows takes 2.2 us instead of 2.45, and to make one takes 0.013 us a tile of the machine's time; so it pays from about four blocks of rows
// to a tile on.  Not beyond a gigabyte, as a cache in 4 bits is there for want of memory.
int64_t image_bytes(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int group) {
  int64_t tiles = 0, blocks = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t t = seqs[i].count > 0 ? ceil_div(seqs[i].length, kKeyTile) : 0;
    tiles += t, blocks += t * ceil_div((int64_t)seqs[i].count * group, kBlockRows);
  }
  const int64_t bytes = tiles * c->n_kv_heads * 2 * kKeyTile * c->head_dim * 2;
  return blocks >= 4 * tiles && bytes <= 1 << 30 ? bytes + ceil_div(tiles * c->n_kv_heads * 4, 16) * 16 : 0;
}

// the units of the attention of seqs[0 .. n - 1] for many rows
int lay_out_many(const infllm_packed* c, const infllm_packed_seq* seqs, int n_sm, PackedTcParams& P, bool* join) {
  const int group = P.a.group;
  INFLLM_TRY(many_units(c, seqs, P, [](const infllm_packed_seq& s, int g) { return (int)ceil_div((int64_t)s.count * g, kBlockRows); }));
  deal_out(P, n_sm, join, [&](auto&& f) {
    for (int i = 0; i < P.a.batch; ++i)
      for (int h = 0; h < c->n_kv_heads && seqs[i].count > 0; ++h)
        for (int x = 0; x < P.a.seq[i].chunks; ++x) f(tiles_of(P.a.seq[i], group, x), tile_work(std::min<int64_t>(kBlockRows, (int64_t)seqs[i].count * group - (int64_t)x * kBlockRows)));
  });
  return INFLLM_OK;
}

// and of their weights
int lay_out_weights(const infllm_packed* c, const infllm_packed_seq* seqs, int n_sm, PackedTcParams& P, bool* join) {
  INFLLM_TRY(many_units(c, seqs, P, [](const infllm_packed_seq& s, int) { return s.count > 0 ? (int)ceil_div(s.length, kWeighKeys) : 0; }));
  deal_out(P, n_sm, join, [&](auto&& f) {
    for (int i = 0; i < P.a.batch; ++i)
      for (int h = 0; h < c->n_kv_heads && seqs[i].count > 0; ++h)
        for (int x = 0; x < P.a.seq[i].chunks; ++x) f(weigh_tiles(P.a.seq[i], P.a.group, P.a.weigh, x), 2);
  });
  return INFLLM_OK;
}

int check_attend(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int most, int n_heads, int weigh, int64_t* bytes, const char* what) {
  INFLLM_TRY(packed_check(c, what));
  INFLLM_TRY(packed_check_seqs(c, seqs, n, most, what));
  if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads > 1 << 16) return fail(INFLLM_E_BADARG, "%s: %d query heads over %d KV heads", what, n_heads, c->n_kv_heads);
  if (weigh < 0) return fail(INFLLM_E_BADARG, "%s: the weights of %d tokens", what, weigh);
  if ((int64_t)most * n_heads > INT_MAX / 4) return fail(INFLLM_E_BADARG, "%s: %d tokens of %d heads", what, most, n_heads);
  *bytes = 0;
  if (n == 0 || most == 0) return INFLLM_OK;
  const int n_sm = sm_count(c->device);
  const int group = n_heads / c->n_kv_heads;
  if (many_rows(seqs, n, group)) {
    int64_t image = 0;
    for (int b0 = 0; b0 < n; b0 += kAttnSeqs) image = std::max(image, image_bytes(c, seqs + b0, std::min(n - b0, kAttnSeqs), group));
    *bytes = image + (int64_t)2 * n_sm * kBlockRows * (c->head_dim + 1) * 4 + (weigh > 0 ? (int64_t)n * most * n_heads * 4 : 0);
    return INFLLM_OK;
  }
  int64_t units = 0;
  PackedAttnSeq to[kAttnSeqs];
  bool join = false;
  for (int b0 = 0; b0 < n; b0 += kAttnSeqs) units = std::max(units, lay_out_few(c, seqs + b0, std::min(n - b0, kAttnSeqs), n_sm, to, &join));
  const int64_t sums = weigh > 0 ? std::min(n, kAttnSeqs) * (int64_t)c->n_kv_heads * (logit_pitch(seqs, n) / kSumKeys) : 0;  // (blocks of a launch)
  if (units > INT_MAX || sums > INT_MAX / 2) return fail(INFLLM_E_BADARG, "%s: %lld units of work, the weights of %lld thousand tokens", what, (long long)units, (long long)sums);
  *bytes = ceil_div(units * c->n_kv_heads * kFewRows * (c->head_dim + 1) * 4, 16) * 16 + (weigh > 0 ? (int64_t)n * most * n_heads * logit_pitch(seqs, n) * 4 : 0);
  return INFLLM_OK;
}

int n_heads_of(const PackedAttnParams& P) { return P.at.n_kv * P.group; }

template <typename T, int kDim>
int attend_few(PackedAttnParams& P, const infllm_packed_seq* seqs, const infllm_packed* c, int n_sm, bool join, cudaStream_t s) {
  const int64_t units = lay_out_few(c, seqs, P.batch, n_sm, P.seq, &join);
  int counts = 0;
  for (int i = 0; i < P.batch; ++i) counts = std::max(counts, seqs[i].count);
  P.part_lse = P.part_o + units * c->n_kv_heads * kFewRows * kDim;
  if (units > 0) {
    auto kern = counts * P.group <= 4 ? (P.logits ? packed_rows_kernel<T, kDim, true, true> : packed_rows_kernel<T, kDim, true, false>)
                                      : (P.logits ? packed_rows_kernel<T, kDim, false, true> : packed_rows_kernel<T, kDim, false, false>);
    INFLLM_CUDA_OK(launch_chained(kern, dim3((unsigned)units, c->n_kv_heads), dim3(kAttnWarps * 32), 0, s, P));
    INFLLM_LAUNCH_OK("packed_rows_kernel");
  }
  if (!join && (!P.logits || units == 0)) return INFLLM_OK;
  const int64_t rows = (int64_t)P.batch * P.most * n_heads_of(P);
  return by_warps(rows, n_sm, [&](auto warps) {
    constexpr int kWarps = decltype(warps)::value;
    P.join_blocks = join ? (int)ceil_div(rows * kWarps, 8) : 0;
    const int64_t sums = P.logits ? (int64_t)P.batch * P.at.n_kv * (P.pitch / kSumKeys) : 0;
    return launch_chained(packed_join_kernel<T, kDim, kWarps>, dim3((unsigned)(P.join_blocks + sums)), dim3(256), 0, s, P);
  });
}

template <typename T, int kDim>
int attend_many(PackedTcParams& P, const infllm_packed_seq* seqs, const infllm_packed* c, char* work, int n_sm, cudaStream_t s) {
  const int64_t image = image_bytes(c, seqs, P.a.batch, P.a.group);
  bool cut = false;
  INFLLM_TRY(lay_out_many(c, seqs, n_sm, P, &cut));
  P.image = image > 0 ? work : nullptr, P.n_image = 0;
  int fewest = P.a.most, rows = 0;
  for (int i = 0; i < P.a.batch; ++i) {
    P.a.seq[i].keys = P.n_image;
    if (image > 0 && seqs[i].count > 0) P.n_image += c->n_kv_heads * (int)ceil_div(seqs[i].length, kKeyTile);  // (up to 16384, in a gigabyte)
    fewest = std::min(fewest, seqs[i].count), rows = std::max(rows, std::min(kBlockRows, seqs[i].count * P.a.group));
  }
  P.odd = (int32_t*)(work + (int64_t)P.n_image * 2 * kKeyTile * kDim * 2);
  P.a.part_o = (float*)(work + image), P.a.part_lse = P.a.part_o + (int64_t)2 * n_sm * kBlockRows * kDim;
  INFLLM_TRY(tc_get_error_ptr(&P.a.err));
  if (P.n_ctas > 0) INFLLM_TRY(packed_tc_launch(P, c->dtype, kDim, s));
  if (cut)
    INFLLM_TRY(by_warps((int64_t)P.n_ctas * rows, n_sm, [&](auto warps) {
      constexpr int kWarps = decltype(warps)::value;
      return launch_chained(packed_join_cut_kernel<T, kDim, kWarps>, dim3((unsigned)ceil_div(rows * kWarps, 8), P.n_ctas), dim3(256), 0, s, P);
    }));
  if (fewest < P.a.most) {
    INFLLM_CUDA_OK(launch_chained(packed_empty_kernel<T, kDim>, dim3((unsigned)ceil_div((int64_t)(P.a.most - fewest) * n_heads_of(P.a), 8), P.a.batch), dim3(256), 0, s, P.a));
    INFLLM_LAUNCH_OK("packed_empty_kernel");
  }
  return INFLLM_OK;
}

}  // namespace

}  // namespace infllm

using namespace infllm;

extern "C" int infllm_packed_room(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int most, int n_heads, int weigh, int64_t* work_bytes) {
  return guarded("packed_room", [&]() -> int {
    if (!work_bytes) return fail(INFLLM_E_BADARG, "packed_room: null pointer");
    return check_attend(c, seqs, n, most, n_heads, weigh, work_bytes, "packed_room");
  });
}

extern "C" int infllm_packed_attend(const infllm_packed* c, int layer, const infllm_packed_seq* seqs, int n, int most, const void* d_q,
                                    int64_t q_bs, int64_t q_hs, int64_t q_ts, void* d_out, float* d_lse, int n_heads, float scale, int weigh,
                                    float decay, void* d_work, int64_t work_bytes, void* stream) {
  return guarded("packed_attend", [&]() -> int {
    int64_t bytes = 0;
    INFLLM_TRY(check_attend(c, seqs, n, most, n_heads, weigh, &bytes, "packed_attend"));
    if (layer < 0 || layer >= c->n_layers) return fail(INFLLM_E_BADARG, "packed_attend: layer %d of %d", layer, c->n_layers);
    if (!(scale >= 0.f) || !std::isfinite(scale * kLog2e)) return fail(INFLLM_E_BADARG, "packed_attend: a scale of %g", (double)scale);
    if (!(decay >= 0.f) || !std::isfinite(decay)) return fail(INFLLM_E_BADARG, "packed_attend: a decay of %g", (double)decay);
    if (n == 0 || most == 0) return INFLLM_OK;
    if (!d_q || !d_out) return fail(INFLLM_E_BADARG, "packed_attend: null pointer");
    if (((uintptr_t)d_q | (uintptr_t)d_out) % 16 || (q_bs | q_hs | q_ts) % 8) return fail(INFLLM_E_BADARG, "packed_attend: rows must be 16-byte aligned");
    if (work_bytes < bytes || (bytes > 0 && (!d_work || (uintptr_t)d_work % 16)))
      return fail(INFLLM_E_BADARG, "packed_attend: a workspace of %lld bytes, 16-byte aligned", (long long)bytes);
    DeviceScope scope(c->device);
    cudaStream_t s = (cudaStream_t)stream;
    PackedTcParams Tc;
    PackedAttnParams& P = Tc.a;
    P.at = packed_planes(c, layer);
    P.q = (const char*)d_q, P.q_bs = q_bs * 2, P.q_hs = q_hs * 2, P.q_ts = q_ts * 2;
    P.out = (char*)d_out, P.lse = d_lse;
    const bool many = many_rows(seqs, n, n_heads / c->n_kv_heads);
    P.pitch = logit_pitch(seqs, n), P.logit_rows = most * (n_heads / c->n_kv_heads);
    // (what the weights are worked out of, at the end of the workspace)
    P.logits = weigh > 0 && !many ? (float*)((char*)d_work + bytes - (int64_t)n * most * n_heads * P.pitch * 4) : nullptr;
    P.row_lse = weigh > 0 && many ? (float*)((char*)d_work + bytes - (int64_t)n * most * n_heads * 4) : nullptr;
    P.weights = c->d_weights + layer * packed_rows(c);
    P.part_o = (float*)d_work;
    P.group = n_heads / c->n_kv_heads, P.most = most, P.weigh = weigh;
    // (the tensor-core kernel masks scores before it scales them: -inf times 0 is no number.  By the least normal number instead, scores
    // of less than 2^100 are zeros beside any reference)
    P.scale_log2 = std::max(scale * kLog2e, FLT_MIN), P.decay = decay;
    const int n_sm = sm_count(c->device);
    for (P.b0 = 0; P.b0 < n; P.b0 += kAttnSeqs) {
      P.batch = std::min(n - P.b0, kAttnSeqs);
      const infllm_packed_seq* mine = seqs + P.b0;
      int64_t longest = 0;
      bool empty = false, any = false;  // rows without a token, rows with one
      for (int i = 0; i < P.batch; ++i) {
        if (mine[i].count > 0) longest = std::max<int64_t>(longest, mine[i].length), any = true;
        empty = empty || mine[i].count < most;
      }
      INFLLM_DISPATCH_DTYPE(c->dtype, T, {
        if (many) INFLLM_TRY((c->head_dim == 128 ? attend_many<T, 128>(Tc, mine, c, (char*)d_work, n_sm, s) : attend_many<T, 64>(Tc, mine, c, (char*)d_work, n_sm, s)));
        else INFLLM_TRY((c->head_dim == 128 ? attend_few<T, 128>(P, mine, c, n_sm, empty, s) : attend_few<T, 64>(P, mine, c, n_sm, empty, s)));
        if (weigh > 0 && any && many) {
          bool cut = false;
          INFLLM_TRY(lay_out_weights(c, mine, n_sm, Tc, &cut));
          INFLLM_TRY(packed_weigh_tc_launch(Tc, c->dtype, c->head_dim, cut, (int)longest, s));
        }
      });
    }
    return INFLLM_OK;
  });
}
