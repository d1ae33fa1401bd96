// What the kernels of the attention over the cache in 4 bits are given (packed_attn.cu, packed_tc.cu).
#pragma once
#include "packed.cuh"

namespace infllm {

constexpr int kAttnSeqs = 128;  // of a launch
constexpr int kBlockRows = 256, kKeyTile = 128;  // of the tensor-core kernels
constexpr int kMaxSms = 160;

// The reference of a row's exponentials, p = 2^(s - reference), is lazy: it moves where the maximum is more than kGrow above it, to kBelow under
// the maximum, so that p is 2^kGrow at most, and the largest 2^kBelow or more.  fp16 has no numbers below 2^-24, and only a few digits
// below 2^-14: its reference is as low as its largest numbers allow, or what many keys together have beside one (a first token that
// takes nearly all attention) would be lost from the products and not from the sums.
template <typename T>
struct Reference {
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  static constexpr float kGrow = kBf16 ? 8.f : 15.f, kBelow = kBf16 ? 0.f : 11.f;
};

struct PackedAttnSeq {
  int32_t slot, length, count;
  int32_t unit0;   // its first unit of work, and how they follow from there:
  int32_t chunks;  // few rows: unit0 + stretch of `keys` keys
  int32_t keys;    // many: unit0 + KV head * chunks + block of 256 rows; its first tile of the image
};

struct PackedAttnParams {
  PackedPlanes at;
  const char* q;
  int64_t q_bs, q_hs, q_ts;  // bytes
  char* out;
  float* lse;
  float *part_o, *part_lse;  // few rows: 8 of each unit and KV head; many: kBlockRows rows of each block's first and last unit
  float* row_lse;            // (batch, KV head, token, query head of the KV head), to base 2: for the weights; null: none
  float* weights;            // of the layer
  float* logits;             // (batch, KV head, row, pitch): scores to base 2 of up to 8 rows, for the weights; null: none
  int64_t pitch;
  int32_t logit_rows, join_blocks;  // blocks of the join; those behind them add up the weights
  int* err;
  int32_t group, most, batch, b0, weigh;
  float scale_log2, decay;
  PackedAttnSeq seq[kAttnSeqs];
};

// Many rows: the key tiles of all units, one unit behind the other, are dealt out to the blocks in stretches of about equal work; block c
// has those from start[c] to start[c + 1], as (unit, tile).
struct PackedTcParams {
  PackedAttnParams a;
  int32_t n_ctas, n_image;
  char* image;  // prompts: n_image tiles, keys and values, as 16-bit numbers (packed_tc.cu); null: none
  int32_t* odd;  // of each, behind it, a multiple of 4 words: whether it has 0 where a value is no number
  int2 start[kMaxSms + 1];
};

// the launch's sequence that has unit u (of several that begin there, those without units come first)
__device__ __forceinline__ int seq_of(const PackedAttnParams& P, int u) {
  int lo = 0, hi = P.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (P.seq[mid].unit0 <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// keys that row r of a sequence's new tokens sees
__host__ __device__ __forceinline__ int keys_of_row(const PackedAttnSeq& S, int group, int r) { return S.length - S.count + r / group + 1; }
// key tiles of a block of rows
__host__ __device__ __forceinline__ int tiles_of(const PackedAttnSeq& S, int group, int block) {
  const int rows = S.count * group, last = block * kBlockRows + kBlockRows - 1;
  return (keys_of_row(S, group, last < rows ? last : rows - 1) + kKeyTile - 1) / kKeyTile;
}

// the weights, for many rows: units of 256 keys of a KV head (unit0 + KV head * chunks + block) by tiles of 128 counted rows that see them
constexpr int kWeighKeys = 256;
__host__ __device__ __forceinline__ int weigh_row0(const PackedAttnSeq& S, int group, int weigh, int block) {
  const int counted = S.count - (weigh < S.count ? weigh : S.count), sees = block * kWeighKeys - (S.length - S.count);
  return (counted > sees ? counted : sees) * group;
}
__host__ __device__ __forceinline__ int weigh_tiles(const PackedAttnSeq& S, int group, int weigh, int block) {
  return (S.count * group - weigh_row0(S, group, weigh, block) + 127) / 128;
}

#ifdef __CUDACC__
// the last block whose stretch begins at or before (unit, tile)
__device__ __forceinline__ int block_of(const PackedTcParams& P, int u, int t) {
  int lo = 0, hi = P.n_ctas - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (P.start[mid].x < u || (P.start[mid].x == u && P.start[mid].y <= t)) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// the 32 numbers of a group, codes c and (m, s), to row k of a swizzled tile; `to` is the tile's half that has group t
template <typename T>
__device__ __forceinline__ void put_group(unsigned char* to, int k, int t, const uint4& c, uint32_t ms) {
  using C = Codes<T>;
  const auto m2 = C::least2(ms), s2 = C::step2(ms);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // (the 16 bytes of eight lanes at a time go to eight different bank groups: lanes of the second half of a row are two pieces ahead)
    const int at = j ^ (t >> 1) * 2;
    const uint32_t x = t >> 1 ? w[j ^ 2] : w[j];
    uint32_t v[4];
    C::pairs(x, m2, s2, v);
    *reinterpret_cast<uint4*>(to + k * 128 + ((((t & 1) * 4 + at) ^ (k & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}
#endif

int packed_weigh_tc_launch(const PackedTcParams& P, int dtype, int head_dim, bool join, int longest, cudaStream_t s);
int packed_tc_launch(const PackedTcParams& P, int dtype, int head_dim, cudaStream_t s);

}  // namespace infllm
