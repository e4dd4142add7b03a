// A paged cache of keys and values held as e4m3 codes.
//
// A page holds, for every cache of its group, keys then values, each [kv_heads][page_tokens][head_dim] codes; beside the pages
// lie the scales, per page and cache keys' then values', each [kv_heads][page_tokens / SCALE_TOKENS] float32.  The number that a
// code stands for is code * scale.  What the format keeps, and every kernel here counts on:
//  - a scale is a power of two, 2^e with SCALE_LEAST <= e <= SCALE_MOST: code * scale is then exactly a bfloat16 (four bits of
//    a bfloat16's eight, and its range), and a scale can grow without rounding the codes that it covered (but for those that fall
//    below e4m3's normal range);
//  - e is the smallest with 448 * 2^e no less than the block's largest entry in size;
//  - codes are finite.  A block of SCALE_TOKENS positions that was given a NaN or an infinity, as key or value, has NaN as its keys'
//    scale: every query that sees one of its keys gets NaN, a query to which all of them are hidden none.
#pragma once

#include "common.cuh"

constexpr int SCALE_TOKENS = 16;
constexpr int SCALE_LEAST = -100, SCALE_MOST = 119;

struct Cache8 {
  uint8_t* k;                  // this cache's part of page 0
  uint8_t* v;
  float* k_scale;              // this cache's scales of page 0
  float* v_scale;
  const int32_t* block_table;  // [batch sequences][table_stride]: page of a request's n-th block, below zero if none
  long long page_stride;       // codes from one page to the next
  long long scale_stride;      // scales from one page to the next
  int n_pages;                 // of the pool: the table's entries outside 0 .. n_pages - 1 count as no page
  int table_stride;
  int page_tokens;             // a multiple of SCALE_TOKENS
  int kv_heads;
  int head_dim;
};

// What the kernels of a step go by: the arrays of llm_step_maps.
struct StepLists {
  const int32_t *seq_q_start, *seq_q_len, *seq_kv_len;   // per request: first row, new tokens, length after the step
  const int32_t *write_seq, *write_block;                // blocks of SCALE_TOKENS positions that the step writes; -1, 0 behind the last
  const int32_t* order;                                  // the requests, longest first
  const int32_t *tile_seq, *tile_index;                  // tiles of the requests with many rows; -1, 0 behind the last
  int n_seqs, n_writes, n_tiles;
};

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
// The exponent of a normal positive power of two.
__device__ __forceinline__ int exponent_of(float s) { return (__float_as_int(s) >> 23) - 127; }

// The current device's bit in the launchers' record of where a kernel's attributes are set (they hold for one device).
static inline unsigned long long device_bit() {
  int device = 0;
  cudaGetDevice(&device);
  return 1ull << (device & 63);
}

// What a sink (base-2 units) adds to a row's sum against the maximum m, infinite ones and rows without a maximum included.
__device__ __forceinline__ float sink_share(float sink, float m) {
  return sink == -INFINITY ? 0.0f : sink == INFINITY ? INFINITY : exp2f(sink - m);
}

// The page that holds `position` (zero or more) of batch sequence `seq`, -1 if none does.
__device__ __forceinline__ int page_of(const Cache8& c, int seq, int position) {
  const int block = position / c.page_tokens;
  const int page = block < c.table_stride ? __ldg(c.block_table + (long long)seq * c.table_stride + block) : -1;
  return page < c.n_pages ? page : -1;
}
