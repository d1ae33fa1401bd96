// A warp's share of the attention of up to 16 rows of a KV head over the keys of a unit (paged_attn.cu has the formulas): groups
// of 16 keys, keys and values from global memory straight into the registers that are the operands of the m16n8k16 products
// (decode_warp.cuh has the same arrangement for eight rows of 128 dimensions, and says how the fragments follow).
//
// What bounds it is the bytes of the keys and values: a warp has a whole group of them, 4 to 8 KB, on its way at once.
// P is two 16-bit numbers, p = hi + lo, so that an output's only rounding is its own (with one the error against 64 bits is 1.4
// times as large): the second product costs nothing that shows beside the loads.
#pragma once
#include "decode_warp.cuh"
#include "paged_attn.cuh"

namespace infllm {

constexpr int kRowWarps = 4;
constexpr int kRowTile = 16;
// blocks of four warps per SM: as many as 128 or 168 registers a thread leave room for
constexpr int row_blocks(int tiles_of_eight) { return tiles_of_eight > 1 ? 3 : 4; }

template <typename T, int kDim, int kNt>  // kNt: tiles of eight rows
struct RowsWarp {
  static constexpr int kJ = kDim / 32;  // 16-byte pieces of a row that a thread has as scores' operands
  static constexpr int kH = kDim / 64;  // of a value's row
  const char* from[kNt];
  uint4 qf[kNt][kJ];
  int lim[kNt];
  float ot[8][kNt][4];  // O^T: [0], [1] = dimension g*8+i of rows 2t, 2t+1; [2], [3] = dimension 64+g*8+i
  float m[kNt], l[kNt];

  // where this thread's rows are: of the plan alone, so before the kernels before on the stream have ended
  __device__ __forceinline__ void find(const PagedParams& P, const AttnUnit& U, int hkv) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int x = 0; x < kNt; ++x) {
      const int r = x * 8 + g;
      lim[x] = 0, from[x] = nullptr;
      if (r < U.rows) {
        const RowAt a = row_at(P, U.node_seq, U.row0 + r);
        // (a row without a token sees nothing)
        lim[x] = a.i < P.most - __ldg(&P.seq[a.b].count) ? 0 : min(U.lim0 + a.i, U.key0 + U.keys);
        from[x] = P.q + a.b * P.q_bs + (int64_t)(hkv * P.group + a.h) * P.q_hs + a.i * P.q_ts + t * 16;
      }
    }
  }
  __device__ __forceinline__ void begin(const PagedParams& P) {
#pragma unroll
    for (int x = 0; x < kNt; ++x) {
#pragma unroll
      for (int j = 0; j < kJ; ++j) qf[x][j] = from[x] ? __ldg(reinterpret_cast<const uint4*>(from[x] + j * 64)) : make_uint4(0, 0, 0, 0);
      m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ot[i][x][0] = ot[i][x][1] = ot[i][x][2] = ot[i][x][3] = 0.f;
    }
  }

  // the groups first, first + step, .. of a unit.  A lane knows the page of one of the next 32; where the warp is one of few on its
  // SM (kFar) it has the next groups but one brought to L2 by then.
  template <bool kFar>
  __device__ __forceinline__ void groups(const PagedParams& P, const AttnUnit& U, int hkv, int first, int step) {
    const int lane = threadIdx.x & 31, n = (U.keys + 15) / 16;
    const int32_t* row = P.table + (int64_t)U.row * P.max_pages;
    auto where = [&](int id, int it) {
      return P.pages + (((int64_t)id * P.n_kv + hkv) * P.page + (U.key0 + it * 16) % P.page) * (kDim * 2);
    };
#pragma unroll 1
    for (int base = first; base < n; base += 32 * step) {
      const int mine = base + lane * step;
      const int id = mine < n ? __ldg(row + (U.key0 + mine * 16) / P.page) : 0;
      if (kFar && mine < n && lane >= 1 && lane < kAhead) prefetch(P, where(id, mine), min(16, U.keys - mine * 16));
#pragma unroll 1
      for (int k = 0; k < 32 && base + k * step < n; ++k) {
        if (kFar && lane == k + kAhead && mine < n) prefetch(P, where(id, mine), min(16, U.keys - mine * 16));
        group(P, U, base + k * step, where(__shfl_sync(0xffffffffu, id, k), base + k * step));
      }
    }
  }
  static constexpr int kAhead = 4;
  __device__ __forceinline__ void prefetch(const PagedParams& P, const char* kb, int keys) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(kb), "r"(keys * kDim * 2) : "memory");
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(kb + P.plane), "r"(keys * kDim * 2) : "memory");
  }

  __device__ __forceinline__ void group(const PagedParams& P, const AttnUnit& U, int it, const char* kb) {
    using namespace mma;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int j0 = U.key0 + it * 16, nk = min(16, U.key0 + U.keys - j0);
    const char* vb = kb + P.plane;
    uint4 kr[2][kJ], vr[4][kH];
    // (what lies behind the last key is not read: it may not be a number, and 0 times that is none)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int r = nt * 8 + g;
      const char* rp = kb + (r < nk ? r : nk - 1) * (kDim * 2) + t * 16;
#pragma unroll
      for (int j = 0; j < kJ; ++j) kr[nt][j] = ld_stream16(rp + j * 64);
    }
#pragma unroll
    for (int ki = 0; ki < 4; ++ki) {
      const int r = 2 * t + (ki & 1) + (ki >> 1) * 8;
      const char* rp = vb + (r < nk ? r : nk - 1) * (kDim * 2) + g * 16;
#pragma unroll
      for (int j = 0; j < kH; ++j) vr[ki][j] = ld_stream16(rp + j * 128);
    }
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const uint32_t a0[4] = {qf[0][j].x, kNt > 1 ? qf[kNt - 1][j].x : 0u, qf[0][j].y, kNt > 1 ? qf[kNt - 1][j].y : 0u};
        mma16816<T>(s[nt], a0, kr[nt][j].x, kr[nt][j].y);
        const uint32_t a1[4] = {qf[0][j].z, kNt > 1 ? qf[kNt - 1][j].z : 0u, qf[0][j].w, kNt > 1 ? qf[kNt - 1][j].w : 0u};
        mma16816<T>(s[nt], a1, kr[nt][j].z, kr[nt][j].w);
      }
    }
    uint32_t hi[kNt][2], lo[kNt][2];
#pragma unroll
    for (int x = 0; x < kNt; ++x) {  // row x * 8 + g: keys nt * 8 + 2t + e
      float v[4], mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = j0 + (k >> 1) * 8 + 2 * t + (k & 1);
        v[k] = key < lim[x] ? s[k >> 1][x * 2 + (k & 1)] * P.scale_log2 : -INFINITY;
        mx = fmaxf(mx, v[k]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[x], mx), ms = mn == -INFINITY ? 0.f : mn;
      const float al = exp2f(m[x] - ms);
      m[x] = mn;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = exp2f(v[k] - ms);
      l[x] = l[x] * al + (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        typename Act<T>::T2 h = Act<T>::from_f2(v[2 * k], v[2 * k + 1]);
        hi[x][k] = *reinterpret_cast<uint32_t*>(&h);
        const float2 f = Act<T>::to_f2(h);
        lo[x][k] = pack2<T>(v[2 * k] - f.x, v[2 * k + 1] - f.y);
      }
      // this thread's columns of O^T are rows 2t and 2t + 1
      const float a0 = __shfl_sync(0xffffffffu, al, (2 * t) * 4), a1 = __shfl_sync(0xffffffffu, al, (2 * t + 1) * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ot[i][x][0] *= a0;
        ot[i][x][1] *= a1;
        ot[i][x][2] *= a0;
        ot[i][x][3] *= a1;
      }
    }
    const uint32_t* w[4][kH];
#pragma unroll
    for (int ki = 0; ki < 4; ++ki)
#pragma unroll
      for (int j = 0; j < kH; ++j) w[ki][j] = reinterpret_cast<const uint32_t*>(&vr[ki][j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i >> 1;
      const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;  // the high or the low 16 bits of both words
      uint32_t a[4];
      a[0] = __byte_perm(w[0][0][r], w[1][0][r], sel);  // dimension g*8+i of keys 2t, 2t+1
      a[2] = __byte_perm(w[2][0][r], w[3][0][r], sel);  // of keys 2t+8, 2t+9
      a[1] = kH > 1 ? __byte_perm(w[0][kH - 1][r], w[1][kH - 1][r], sel) : 0u;  // dimension 64+g*8+i
      a[3] = kH > 1 ? __byte_perm(w[2][kH - 1][r], w[3][kH - 1][r], sel) : 0u;
#pragma unroll
      for (int x = 0; x < kNt; ++x) {
        mma16816<T>(ot[i][x], a, hi[x][0], hi[x][1]);
        mma16816<T>(ot[i][x], a, lo[x][0], lo[x][1]);
      }
    }
  }

  // the rows' sums, whole in every thread of a row
  __device__ __forceinline__ void sums() {
#pragma unroll
    for (int x = 0; x < kNt; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (l[x] != l[x] && m[x] == -INFINITY) m[x] = 0.f;  // (scores that are no numbers are not seen by the maximum)
    }
  }

  // A unit by one warp alone, which leaves its partial rows.
  __device__ __forceinline__ void alone(const PagedParams& P, const AttnUnit& U, int hkv) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    find(P, U, hkv);
    begin(P);
    groups<true>(P, U, hkv, 0, 1);
    sums();
    const int64_t first = (int64_t)U.part + hkv * U.part_kv;
#pragma unroll
    for (int x = 0; x < kNt; ++x) {
      if (t == 0 && x * 8 + g < U.rows) P.part_lse[first + x * 8 + g] = m[x] == -INFINITY ? -INFINITY : m[x] + log2f(l[x]);
      const float inv = m[x] == -INFINITY ? 0.f : 1.f / l[x];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = x * 8 + 2 * t + e;
        const float f = __shfl_sync(0xffffffffu, inv, (2 * t + e) * 4);
        if (r >= U.rows) continue;
        float* to = P.part_o + (first + r) * kDim + g * 8;
#pragma unroll
        for (int h = 0; h < kH; ++h)
#pragma unroll
          for (int i = 0; i < 8; i += 4)
            *reinterpret_cast<float4*>(to + h * 64 + i) = make_float4(ot[i][x][2 * h + e] * f, ot[i + 1][x][2 * h + e] * f, ot[i + 2][x][2 * h + e] * f, ot[i + 3][x][2 * h + e] * f);
      }
    }
  }
};

}  // namespace infllm
