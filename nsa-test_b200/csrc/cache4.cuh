// The 4-bit paged key/value cache: layout, quantisation and argument blocks shared by its kernels.
//
// A page holds kPageTokens tokens of every kv group; the cache is [pages][groups][page bytes].  A page of one group is four records
// of 16 tokens.  A record holds one chunk of 256 bytes per 32 dimensions (those of the keys, then those of the values), then 16
// scales in fp16 per chunk.  The codes lie as the fragments of mma.m16n8k16 want them, so that a warp reads a chunk with one
// 8-byte load per lane and needs no transposition:
//   keys    lane 4 n + j holds dimensions 8 j + e (nibble e) of token n (word 0) and token 8 + n (word 1)
//   values  lane 4 n + j holds dimensions 8 e + n (nibble e) of tokens 2 j, 2 j + 1, 8 + 2 j, 8 + 2 j + 1 (16 bits each)
//   scales  token 8 t + 2 j + b at place 4 j + 2 t + b: the two words of lane j hold the scales of its four tokens
// Every byte belongs to one token, so tokens of the same record can be written by different threads at once.
//
// A code c stands for (c - 8) s.  s is a seventh of the group's largest magnitude rounded to 8 significant bits, so that every value
// has at most 11 and is exact in fp16: the tensor-core kernels multiply what the cache holds, without a rounding of their own.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace nsa {

constexpr int kPageTokens = 64, kRecTokens = 16, kGroupDims = 32;
constexpr int kChunkBytes = 256, kChunkScaleBytes = 32, kRecBytesPerGroup = kChunkBytes + kChunkScaleBytes;
constexpr int kRecsPerPage = kPageTokens / kRecTokens;
constexpr float kMaxHeld = 57120.f;   // 7 * 8160, 8160 the largest scale of 8 significant bits whose eightfold is finite in fp16

__host__ __device__ __forceinline__ int64_t page_bytes(int dk, int dv) { return (int64_t)kRecsPerPage * ((dk + dv) / kGroupDims) * kRecBytesPerGroup; }

// What the attention kernels need (nsa_cache4_desc with the strides and counts they use).
struct Cache4Args {
  const void* q;
  const uint8_t* cache;
  const int32_t *table, *lengths, *starts, *indices;
  void* out;
  float *L, *M;
  int64_t sq_tok, sq_head, table_ld;
  int N, S, P, H, G, hpg, dk, dv, n_pages, n_sel, window;
  float scale;
  int rows_lo, rows_hi;      // requests with rows_lo <= new * hpg < rows_hi are this launch's
  uint8_t* ws;               // per block: a SplitRecord, then two partial results
};

}  // namespace nsa
