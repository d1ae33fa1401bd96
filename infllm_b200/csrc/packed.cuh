// A key/value cache in 4 bits (packed.cu, packed_attn.cu): what it holds, and how numbers come out of it.
//
// Of each 32 neighbouring numbers x of a row, in the cache's 16-bit type T: the least m, a step s = T((max x - m) / 15), and of each
// number a code c = the nearest of 0 .. 15 to (x - m) / s, ties to even (0 where s is 0).  (Where T(m + 15 s) were infinite, s is the next
// smaller number of T: what the cache stands for is finite wherever m and s are.)  A number stands for T(m + s c): one fused
// multiply-add in T, so every kernel has the same operands, whatever its tiles.
// A word has eight codes, number 2i at bit 4i and number 2i + 1 at bit 16 + 4i: what a mask leaves are two neighbours, and the low or the high halves of two rows' words, put together, give pairs of the same number of both rows.
#pragma once
#include <type_traits>

#include "mma_common.cuh"
#include "pages.cuh"

namespace infllm {

constexpr int kPackGroup = 32;  // numbers that share (m, s)

// the layer's planes and the step between a sequence's heads; rows of a head lie one behind the other
struct PackedPlanes {
  const char* codes;   // keys; values `codes_v` behind them.  A row has kDim / 2 bytes
  const char* scales;  // a row has kDim / 8 bytes: (m, s) of each group
  int64_t codes_v, scales_v;
  int32_t max_tokens, n_kv;
  __device__ __forceinline__ int64_t row0(int slot, int hkv) const { return ((int64_t)slot * n_kv + hkv) * max_tokens; }
};

// A word's codes come out by a mask (and a shift for the upper half of them), a product or a difference that makes them numbers, and one
// multiply-add; the masks and shifts share the slowest pipe, so there are as few of them as can be.
//   bf16  Bits 0 .. 7 of a number are, without its other bits, that whole number times 2^-133 (the first binade goes on where the
//         subnormals end), so codes at bits 0 .. 3 and 4 .. 7 are c and 16 c times 2^-133; a product makes c 2^-6 of both, and the step is
//         64 s.  (A step of 2^122 or more, which has no such product, is not held: its group is NaN.)
//   fp16  Beside the exponent of 1024 they are 1024 + c and 1024 + 16 c.
template <typename T>
struct Codes {
  using T2 = typename Act<T>::T2;
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  static __device__ __forceinline__ T2 as2(uint32_t x) { return *reinterpret_cast<T2*>(&x); }
  static __device__ __forceinline__ uint32_t bits(T2 x) { return *reinterpret_cast<uint32_t*>(&x); }
  // the pairs at bits 4i and 16 + 4i of w, i = 0 .. 3, with least numbers m2 and steps s2
  static __device__ __forceinline__ void pairs(uint32_t w, T2 m2, T2 s2, uint32_t* out) {
    const uint32_t h = w >> 8;
    out[0] = bits(__hfma2(low(w), s2, m2));
    out[1] = bits(__hfma2(high(w), s2, m2));
    out[2] = bits(__hfma2(low(h), s2, m2));
    out[3] = bits(__hfma2(high(h), s2, m2));
  }
  // (m, s) in one word: pairs (m, m) and (s, s), as pairs() wants them
  static __device__ __forceinline__ T2 least2(uint32_t sc) { return as2(__byte_perm(sc, sc, 0x1010)); }
  static __device__ __forceinline__ T2 step2(uint32_t sc) { return scaled(as2(__byte_perm(sc, sc, 0x3232))); }
  // of two rows' words: pairs (m of a, m of b) and (s of a, s of b)
  static __device__ __forceinline__ T2 least2(uint32_t a, uint32_t b) { return as2(__byte_perm(a, b, 0x5410)); }
  static __device__ __forceinline__ T2 step2(uint32_t a, uint32_t b) { return scaled(as2(__byte_perm(a, b, 0x7632))); }
  // whether (m, s) are not both finite: all exponent bits are set in one of them
  static __device__ __forceinline__ bool odd(uint32_t sc) {
    constexpr uint32_t e = kBf16 ? 0x7f80u : 0x7c00u;
    return (sc & e) == e || (sc >> 16 & e) == e;
  }

 private:
  static __device__ __forceinline__ T2 low(uint32_t w) {  // the codes at bits 0 and 16: themselves, or times 2^-6
    if constexpr (kBf16) return __hmul2(as2(w & 0x000f000fu), as2(0x7f007f00u));  // 2^127
    else return __hsub2(as2((w & 0x000f000fu) | 0x64006400u), as2(0x64006400u));
  }
  static __device__ __forceinline__ T2 high(uint32_t w) {  // at bits 4 and 20
    if constexpr (kBf16) return __hmul2(as2(w & 0x00f000f0u), as2(0x7d007d00u));  // 2^123
    else return __hfma2(as2((w & 0x00f000f0u) | 0x64006400u), as2(0x2c002c00u), as2(0xd400d400u));  // times 1/16, less 64
  }
  static __device__ __forceinline__ T2 scaled(T2 s) {
    if constexpr (kBf16) return __hmul2(s, as2(0x42804280u));  // 64
    else return s;
  }
};

// a sequence of a launch
struct PackedSeq {
  int32_t slot, length, count, position;  // tokens, the newest included; the newest; the position of the first of those
};
static_assert(sizeof(PackedSeq) == sizeof(infllm_packed_seq), "");

int packed_check(const infllm_packed* c, const char* what);
int packed_check_seqs(const infllm_packed* c, const infllm_packed_seq* seqs, int n, int most, const char* what);
PackedPlanes packed_planes(const infllm_packed* c, int layer);
inline int64_t packed_rows(const infllm_packed* c) { return (int64_t)c->n_sequences * c->n_kv_heads * c->max_tokens; }  // of a layer

}  // namespace infllm
