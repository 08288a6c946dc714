// Launch interface of the rotary step and of the paged cache's operators (sage_rotary.hip, sage_cache_attn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ksana_sage {

constexpr int kMostAxes = 4;

// x / by for 0 <= x < 2^31 and 1 <= by < 2^31 as a product: by <= 2^n and m = ceil(2^(31 + n) / by), below 2^32, give m x / 2^(31 + n) = x / by + e x / (by 2^(31 + n))
// with 0 <= e < by, an excess below 2^-n <= 1 / by, too little to reach the next whole number.
struct Divisor {
  uint32_t m;
  int shift, by;  // x / by = (m x >> 32) >> shift
};
inline Divisor divisor(int by) {
  int bits = 0;
  while ((INT64_C(1) << bits) < by) ++bits;
  if (bits == 0) return Divisor{0, 0, 1};
  const int s = 31 + bits;
  return Divisor{(uint32_t)(((UINT64_C(1) << s) + by - 1) / by), s - 32, by};
}
__host__ __device__ inline int quotient(int x, const Divisor& d) {
  return d.by == 1 ? x : (int)((uint32_t)(((uint64_t)d.m * (uint32_t)x) >> 32) >> d.shift);
}

// Where the tokens of a batch's sequences lie: token t of entry b in slot t % size of page table[b sB + t / size]
struct PageTable {
  const int32_t* table;
  int64_t sB;
  int width, pages;   // entries of a sequence; pages that exist
  Divisor size;       // tokens of a page
  const int32_t *q_lens, *k_lens;  // new tokens (nullptr: all rows), tokens with the new ones
};

// Rows [B, L, H, D] that a launch takes through
struct RotaryPart {
  const void* src;
  int64_t sB, sL, sH;  // in elements
  void* dst;
  int64_t dB, dL, dH;  // of pages: page, slot and head, in elements, the same of keys and values (other rows are contiguous)
  const float* scale;  // of 8-bit pages: one per head, or nullptr
  int H;
};
struct RotaryParams {
  RotaryPart part[3];  // q and k, which turn, and a cache's values; with a cache keys and values go into pages.  Those without heads take no part
  int B, L, D, R, dtype, interleaved, eight_bits;
  const double* frequencies;  // R / 2 radians per position
  const void* positions;      // nullptr: of the token itself
  int64_t pos_sB, pos_sL, pos_sA;
  int pos64, axes, ends[kMostAxes];  // pairs before ends[a] go by axis a
  float magnitude;
  int inverse;
  PageTable pages;            // table nullptr: no cache
  // filled in by the launcher
  int heads, units, slots, tokens_each, stream;
  Divisor by_heads, by_length;
};
hipError_t launch_rotary(RotaryParams p, hipStream_t s);

struct CacheAttnParams {
  const uint16_t* q;
  uint16_t* o;
  int64_t q_sB, q_sL, q_sH, o_sB, o_sL, o_sH;  // in elements
  const char *k, *v;
  int64_t sP, sS, sH;          // bytes from one page, slot and head to the next, of k and v
  const float *k_scale, *v_scale;  // one per head, or nullptr
  PageTable pages;
  int B, Lq, Hq, Hkv, D, dtype, eight_bits, causal;
  float sm_scale;
  // filled in by the launcher
  int group;                   // Hq / Hkv
  Divisor by_group;
  float c;                     // |sm_scale| log2(e)
  uint32_t flip;               // sign bits of two 16-bit values where sm_scale is negative
  int page_units, slot_units;  // sP and sS in 16 bytes
  int blocks;                  // of query rows of a key head
  int whole, cut, runs;        // blocks that a workgroup walks, and those that up to `runs` do
  float* part;                 // [cut, runs, rows of a block, D], then a pair for every row
};
uint64_t cache_attn_scratch(CacheAttnParams p);
hipError_t launch_cache_attn(CacheAttnParams p, void* scratch, hipStream_t s);

}  // namespace ksana_sage
