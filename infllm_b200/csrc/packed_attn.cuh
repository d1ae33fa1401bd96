// What the kernels of the attention over the cache in 4 bits are given (packed_attn.cu, packed_tc.cu).
#pragma once
#include "packed.cuh"

namespace infllm {

constexpr int kAttnSeqs = 128;  // of a launch
constexpr int kBlockRows = 256, kKeyTile = 128;  // of the tensor-core kernels
constexpr int kMaxSms = 160;

struct PackedAttnSeq {
  int32_t slot, length, count;
  int32_t unit0;   // its first unit of work, and how they follow from there:
  int32_t chunks;  // few rows: unit0 + tile of 16 rows * chunks + stretch of `keys` keys
  int32_t keys;    // many: unit0 + KV head * chunks + block of 256 rows
};

struct PackedAttnParams {
  PackedPlanes at;
  const char* q;
  int64_t q_bs, q_hs, q_ts;  // bytes
  char* out;
  float* lse;
  float *part_o, *part_lse;  // few rows: 16 rows of each unit and KV head; many: kBlockRows rows of each block's first and last unit
  float* row_lse;            // (batch, KV head, token, query head of the KV head), to base 2: for the weights; null: none
  float* weights;            // of the layer
  int* err;
  int32_t group, most, batch, b0, weigh;
  float scale_log2, decay;
  PackedAttnSeq seq[kAttnSeqs];
};

// Many rows: the key tiles of all units, one unit behind the other, are dealt out to the blocks in stretches of about equal work; block c
// has those from start[c] to start[c + 1], as (unit, tile).
struct PackedTcParams {
  PackedAttnParams a;
  int32_t n_ctas, pad;
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

int packed_tc_launch(const PackedTcParams& P, int dtype, int head_dim, cudaStream_t s);

}  // namespace infllm
