// Attention of the last tokens of a batch's sequences on all of their keys in a paged cache: o = softmax(c q k^T) v.
//
// Row i of entry b stands at position k_len - n + i, n being the entry's new tokens; causal rows see the keys up to their own position, others all.  Query rows
// of the heads that share a key head are numbered together.  Keys of pages that do not exist are not seen: zeros stand in their
// place, and their weight is zero.
//
// A wave keeps 32 query rows (S^T = k q^T: a lane holds scores of one row) and walks tiles of 64 keys with a running maximum and sum.  Probabilities are rounded to the
// tensors' type where they are multiplied with the values, as the matrix instructions want them: off by 2^-8 (bf16) or 2^-11 (fp16) of each at most, few rows on 16-bit caches,
// which have them in two parts, by 2^-16 or 2^-22; in fp16 besides by 2^-31 of the row's largest, the half step of its smallest numbers (2^-24, of weights scaled by 2^6).  Everything
// else is fp32.
// A tile's pages are looked up by its 64 keys' lanes ahead of its copies.  Of 8-bit caches the tiles are widened, exactly, on their way to LDS; the scales go into c and into
// the result.  Loops of few blocks are cut into runs, which a second launch joins: a block's runs share the tiles that its sequence really has.
//
// Many rows are bound by the power that the matrix pipes draw: 4096 causal rows on 32768 keys of 128 channels, 40 heads on 8, take 2.32 to 2.40 ms by the card, 1.07 to
// 1.11e15 operations /s, of zeros 1.70.  (The same kernel on keys in a row takes 3 % less; a library's product reaches 1.35e15.)  Few rows are bound by the keys' and values' bytes: one token of 40
// heads on 32760 keys 28.5 us from memory, 4.7 TB/s, and 4 for the join; 64 of up to 8192 tokens 216, 5.5 TB/s.
#include "sage_cache.h"
#include "sage_train_device.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace ksana_sage {

namespace {

extern __shared__ __align__(1024) char cache_lds[];
__device__ __forceinline__ unsigned lds_base() { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)cache_lds; }

constexpr int kCacheBlock = 128;  // query rows of a workgroup
constexpr int kMostRuns = 64, kLeastTiles = 2;
constexpr float kLog2e = 1.44269504088896340736f;
// fp16 probabilities relative to a row's largest lose bits from 2^-14 on: scaled up by 2^6 a factor of 2^6 later.  The reference point lags behind the row's maximum by
// at most 2^kLazy.
constexpr float kLazy = 8.0f;
template <int DT>
constexpr float kShift = DT == KSANA_SAGE_FP16 ? 6.0f : 0.0f;

__device__ const uint4 kZeroRow[16] = {};  // what stands in a missing key's place

struct Extent {
  int rows, keys, first;  // query rows that take part (over the heads of a key head), keys, position of the first new token
};
__device__ __forceinline__ Extent extent_of(const CacheAttnParams& p, int b) {
  int n = p.Lq, keys = p.pages.width * p.pages.size.by;
  take_counts(p.pages.q_lens, p.pages.k_lens, b, n, keys);
  return Extent{keys > 0 ? n * p.group : 0, keys, keys - n};
}
__device__ __forceinline__ int position_of(const CacheAttnParams& p, int row) { return quotient(row, p.by_group); }
__device__ __forceinline__ int keys_seen(const CacheAttnParams& p, const Extent& e, int row) {
  return p.causal ? min(e.keys, e.first + position_of(p, row) + 1) : e.keys;
}

// What a workgroup works on: a key head, a block of its rows and a run of the block's tiles
struct Place {
  int bh, block, run, cut;  // cut: number of the block among those that are cut; -1: a whole block
};

// A block's runs: what each of them walks, and how many there are (one at least)
struct Run {
  int from, to, runs;
};
__device__ __forceinline__ Run run_of(const CacheAttnParams& p, const Extent& e, const Place& place) {
  const int row0 = place.block * kCacheBlock, run = place.run;
  const bool one = place.cut < 0 || p.runs == 1;
  const int keys = row0 < e.rows ? keys_seen(p, e, min(row0 + kCacheBlock, e.rows) - 1) : 0;
  const int tiles = (max(keys, 0) + kTrainTile - 1) / kTrainTile, each = one ? tiles : max(kLeastTiles, (tiles + p.runs - 1) / p.runs);
  return Run{min(run * each, tiles), min((run + 1) * each, tiles), one ? 1 : max(1, (tiles + each - 1) / each)};
}
// Of consecutive workgroups, which land on consecutive XCDs, each has another head: where the heads are a multiple of eight, an XCD keeps its heads' keys to
// itself.  The last blocks, which see the most, come first.
__device__ __forceinline__ Place block_place(const CacheAttnParams& p, int i) {
  const int heads = p.B * p.Hkv, block = i / heads;
  return Place{i - block * heads, p.blocks - 1 - block, 0, -1};
}
__device__ __forceinline__ Place place_of(const CacheAttnParams& p, int at) {
  if (at < p.whole) return block_place(p, at);
  const int run = (at - p.whole) / p.cut, cut = at - p.whole - run * p.cut;
  Place place = block_place(p, p.whole + cut);
  place.run = run;
  place.cut = cut;
  return place;
}

// Key t 64 + lane of the sequence: the entry of its page is on its way, then where it lies
struct Lookup {
  int entry, slot;
  __device__ __forceinline__ void start(const PageTable& pages, const int32_t* table, int t, int keys, int lane) {
    const int key = t * kTrainTile + lane, number = quotient(key, pages.size);
    slot = key - number * pages.size.by;
    entry = -1;
    if (key < keys) entry = table[number];
  }
};
struct Tile64 {
  unsigned at;     // of the lane's key, 16-byte units from the cache's start; all ones: there is none
  uint64_t exist;  // the keys that do
  // Runs of 16 are (aligned ones, of the tile's 64)
  __device__ __forceinline__ bool in_sixteens(const CacheAttnParams& p) const { return p.pages.size.by % 16 == 0 && exist == ~UINT64_C(0); }
  // All 64 there, a slot apart.  (Of pages of 64 slots and more a tile has two at most: if its ends lie 63 slots apart, so does all between.)
  __device__ __forceinline__ bool in_a_row(const CacheAttnParams& p) const {
    return p.pages.size.by >= kTrainTile && exist == ~UINT64_C(0) &&
           (unsigned)__builtin_amdgcn_readlane((int)at, 63) - (unsigned)__builtin_amdgcn_readfirstlane((int)at) == 63u * (unsigned)p.slot_units;
  }
  __device__ __forceinline__ void finish(const CacheAttnParams& p, const Lookup& l) {
    const bool is = (unsigned)l.entry < (unsigned)p.pages.pages;
    at = is ? (unsigned)l.entry * (unsigned)p.page_units + (unsigned)l.slot * (unsigned)p.slot_units : ~0u;
    exist = __ballot(is);
  }
};

// Copies of a tile, the wave's share.  One whose keys lie in a row is one address and a lane offset.  Otherwise a lane's rows of all copies are of 16 neighbours
// (Tile::row_of): where those lie in a row, they are an address of the lane's own and constants.  Elsewhere every copy is looked up.
// (Chunk of 4096 rows on 32768 keys, 40 heads on 8: 2340 us in pages of 64, 2500 in pages of 16, 2630 in pages of 20.)
template <int D, int kWaves>
struct PagedCopy {
  using T = Tile<D>;
  static constexpr int kCopies = T::kCopies / kWaves;
  const char* base;
  unsigned whole;
  __device__ __forceinline__ PagedCopy(const CacheAttnParams& p, const char* cache, int hk, int wave, int lane)
      : base(cache + hk * p.sH), whole((unsigned)T::row_of(wave, lane) * (unsigned)p.sS + lane % T::kPieces * 16) {}
  __device__ __forceinline__ const char* from(unsigned at, int lane) const {
    return (at == ~0u ? reinterpret_cast<const char*>(kZeroRow) : base + (uint64_t)at * 16) + lane % T::kPieces * 16;
  }
  __device__ __forceinline__ void start(const CacheAttnParams& p, const Tile64& keys, unsigned tile, int wave, int lane) const {
    if (keys.in_a_row(p)) {
      const char* first = base + (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane(keys.at) * 16;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) lds_copy16_at(first + T::row_of(c * kWaves, 0) * p.sS, whole, tile + T::copy_at(c * kWaves + wave));
    } else if (keys.in_sixteens(p)) {
      const char* own = from((unsigned)__shfl((int)keys.at, T::row_of(wave, lane)), lane);
#pragma unroll
      for (int c = 0; c < kCopies; ++c) lds_copy16_from(own + T::row_of(c * kWaves, 0) * p.sS, tile + T::copy_at(c * kWaves + wave));
    } else {
#pragma unroll
      for (int c = 0; c < kCopies; ++c)
        lds_copy16_from(from((unsigned)__shfl((int)keys.at, T::row_of(c * kWaves + wave, lane)), lane), tile + T::copy_at(c * kWaves + wave));
    }
  }
};

// A tile of 8-bit rows, the wave's share, on its way through registers: sixteen channels at an access, D / 16 lanes to a row.  (Where an address is the cache's or kZeroRow's the compiler
// makes loads of any address space of both, which count as LDS accesses too: a wait for LDS behind `start` is one for them.  Rows' 16 bytes are written every 32, where lanes of
// neighbouring rows meet in the same banks, 8 cycles for each write.)
template <int DT, int D, int kWaves>
struct WideCopy {
  using T = Tile<D>;
  static constexpr int kPieces = D / 16, kRows = 64 / kPieces, kCopies = kTrainTile / (kRows * kWaves);
  const char* base;
  unsigned whole;
  uint4 raw[kCopies];
  __device__ __forceinline__ WideCopy(const CacheAttnParams& p, const char* cache, int hk, int wave, int lane)
      : base(cache + hk * p.sH), whole((unsigned)(kRows * wave + lane / kPieces) * (unsigned)p.sS + lane % kPieces * 16) {}
  __device__ __forceinline__ void start(const CacheAttnParams& p, const Tile64& keys, int wave, int lane) {
    if (keys.in_a_row(p)) {
      const char* first = base + (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane(keys.at) * 16;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) raw[c] = *reinterpret_cast<const uint4*>(first + kRows * kWaves * c * p.sS + whole);
      return;
    }
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const unsigned at = (unsigned)__shfl((int)keys.at, kRows * (c * kWaves + wave) + lane / kPieces);
      raw[c] = *reinterpret_cast<const uint4*>((at == ~0u ? reinterpret_cast<const char*>(kZeroRow) : base + (uint64_t)at * 16) + lane % kPieces * 16);
    }
  }
  // (exact: e4m3 numbers are numbers of both types)
  static __device__ __forceinline__ v4i widened(unsigned lo, unsigned hi) {
    if constexpr (DT == KSANA_SAGE_BF16)
      return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
    else
      return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))};
  }
  __device__ __forceinline__ void finish(unsigned tile, int wave, int lane) const {
    typedef __attribute__((address_space(3))) v4i* Lds;
    const unsigned lane_at = tile + T::at(kRows * wave + lane / kPieces) + lane % kPieces * 32;  // (T::at is a sum over a row's bits)
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      *(Lds)(uintptr_t)(lane_at + T::at(kRows * kWaves * c)) = widened(raw[c].x, raw[c].y);
      *(Lds)(uintptr_t)(lane_at + T::at(kRows * kWaves * c) + 16) = widened(raw[c].z, raw[c].w);
    }
  }
};

// A lane's query row as B operands: channels 16 s + 8 hh ..
template <int D>
__device__ __forceinline__ void load_row(const uint16_t* row, int hh, uint32_t flip, v4i (&out)[Tile<D>::kSteps]) {
#pragma unroll
  for (int s = 0; s < Tile<D>::kSteps; ++s) {
    const uint4 x = *reinterpret_cast<const uint4*>(row + 16 * s + 8 * hh);
    out[s] = v4i{(int)(x.x ^ flip), (int)(x.y ^ flip), (int)(x.z ^ flip), (int)(x.w ^ flip)};
  }
}
// The lane's row is here from now on: without this the compiler waits for every load under way where its values are used.
template <int N>
__device__ __forceinline__ void row_ready(v4i (&row)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(row[s]));
}
// Accumulator i of 32-key block h is key 32 h + acc_row(i) + 4 hh
__device__ __forceinline__ constexpr int acc_row(int i) { return 8 * (i >> 2) + (i & 3); }

// Scores of keys that the lane's row does not see: `limit` of the tile's, and those of no page.  The largest of the others.
__device__ __forceinline__ float hide_scores(v16f (&s)[2], int limit, uint64_t exist) {
  const int left = max(limit, 0);
  const uint64_t of_tile = left < kTrainTile ? exist & ((UINT64_C(1) << left) - 1) : exist;
  const uint64_t seen = __builtin_amdgcn_inverse_ballot_w64(UINT64_C(0xffffffff) << 32) ? of_tile >> 4 : of_tile;  // (by hh, which would be kept through the loop for it)
  uint32_t bits[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
  pin(bits[0]);  // (a branch that stays one: 64 instructions for every tile otherwise)
  pin(bits[1]);
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) s[h][i] = bits[h] & (1u << acc_row(i)) ? s[h][i] : -INFINITY;
    most = largest(most, s[0][i], s[1][i]);
  }
  return most;
}

// Many rows: four waves of 32 share a tile's copies, two workgroups to a compute unit, so that each SIMD has two waves.  While the probabilities of tile t are formed and
// multiplied with its values, the scores of tile t + 1 are: a few vector instructions stand behind every matrix instruction and run beside it.  So values are
// wanted a step after their keys; each have two places in LDS.  Of 128 channels about 20 registers go through memory, outside the loop.
// 4096 causal rows on 32768 keys, 40 heads on 8, on one card: bf16 2330 us, fp16 2500, 8 bits 2510 (fp16 2600); of 64 channels, 32 heads on 8, 1200, where exponentials count
// twice as much.
template <int DT, int D, bool kEight>
__global__ __launch_bounds__(256, 2) void sage_cache_rows_kernel(const CacheAttnParams p) {
  using T = Tile<D>;
  constexpr int kWaves = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, hh = lane >> 5;
  const int all_rows = p.Lq * p.group;
  const Place place = place_of(p, (int)blockIdx.x);
  const int b = place.bh / p.Hkv, hk = place.bh - b * p.Hkv, row0 = place.block * kCacheBlock;
  const Extent e = extent_of(p, b);
  const Run range = run_of(p, e, place);
  if (place.run >= range.runs) return;

  const unsigned lds = lds_base();
  const float scale = fmaxf(p.c * (p.k_scale != nullptr ? p.k_scale[hk] : 1.0f), 1.2e-38f);  // (times -infinity, where a score is hidden, still that)
  v16f acc[T::kBlocks];
#pragma unroll
  for (int d = 0; d < T::kBlocks; ++d) acc[d] = v16f{};
  float top = -INFINITY, minus = kShift<DT>, sum = 0.0f;  // reference point (unscaled), what is added to scaled scores, the row's sum
  const int row = row0 + wave * 32 + m;
  if (range.from < range.to) {
    using Copy = std::conditional_t<kEight, WideCopy<DT, D, kWaves>, PagedCopy<D, kWaves>>;
    Copy k_copy(p, p.k, hk, wave, lane), v_copy(p, p.v, hk, wave, lane);
    const int32_t* table = p.pages.table + b * p.pages.sB;
    auto k_tile = [&](int t) { return lds + (t & 1) * T::kBytes; };
    auto v_tile = [&](int t) { return lds + (2 + (t & 1)) * T::kBytes; };
    auto copy_keys = [&](int t, const Tile64& keys) {
      if constexpr (kEight)
        k_copy.start(p, keys, wave, lane);
      else
        k_copy.start(p, keys, k_tile(t), wave, lane);
    };
    auto copy_values = [&](int t, const Tile64& keys) {
      if constexpr (kEight)
        v_copy.start(p, keys, wave, lane);
      else
        v_copy.start(p, keys, v_tile(t), wave, lane);
    };
    auto keys_there = [&](int t) {
      if constexpr (kEight) k_copy.finish(k_tile(t), wave, lane);
    };
    auto values_there = [&](int t) {
      if constexpr (kEight) v_copy.finish(v_tile(t), wave, lane);
    };
    // (behind a run's last tile: that one again)
    Lookup next_lookup;
    auto look_up = [&](int t) { next_lookup.start(p.pages, table, min(t, range.to - 1), e.keys, lane); };
    Tile64 here64, next64;  // of this step's tile and the next one
    look_up(range.from);
    here64.finish(p, next_lookup);
    look_up(range.from + 1);
    next64.finish(p, next_lookup);
    copy_keys(range.from, here64);
    look_up(range.from + 2);
    v4i q[T::kSteps];
    {
      const int r = min(row, e.rows - 1), l = position_of(p, r);
      load_row<D>(p.q + b * p.q_sB + l * p.q_sL + (int64_t)(hk * p.group + r - l * p.group) * p.q_sH, hh, p.flip, q);
    }
    const unsigned row_at = row_lane_at<D>(lane), column_at = column_lane_at<D>(lane);
    const int limit = keys_seen(p, e, row);  // keys that the row sees, and that all of the wave see
    const int all_see = keys_seen(p, e, min(row0 + wave * 32, e.rows - 1));
    const bool idle = row0 + wave * 32 >= e.rows;  // a wave without rows copies its share
    float most = -INFINITY;
    auto hide = [&](int t, uint64_t exist, v16f (&s)[2]) {
      if ((t + 1) * kTrainTile <= all_see && exist == ~UINT64_C(0)) return;
      most = hide_scores(s, limit - t * kTrainTile, exist);
    };
    // Tile t: its scores in s, the largest of the lane's in `most`; forms the scores of tile t + 1 in `next` unless `last`.  Its weights are added up by themselves, then to the
    // row's sum: added to that one by one, equal weights are all rounded the same way, 0.34 % of it after 524288 keys.  (Products take 16 keys at an addition.)
    auto compute = [&](int t, v16f (&s)[2], v16f (&next)[2], auto last) {
      const float here = over_halves<Max>(most);
      if (__any(here * scale > kLazy + kShift<DT> - minus || (top == -INFINITY && here > -INFINITY))) {
        const float at = fmaxf(top, here);
        const float factor = top == -INFINITY ? 0.0f : fast_exp2((top - at) * scale);
        top = at;
        minus = at == -INFINITY ? kShift<DT> : kShift<DT> - at * scale;
        sum *= factor;
#pragma unroll
        for (int d = 0; d < T::kBlocks; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] *= factor;
      }
      unsigned k_at = k_tile(t + 1) + row_at, v_at = v_tile(t) + column_at;
      pin(k_at);  // (one address and constants, not sixteen)
      pin(v_at);
      v4i pr[4];
      {
        constexpr int kParts = 2 * T::kSteps, kEach = 32 / kParts, kAhead = kEight ? 2 : 3;  // (8 bits: with three a register of q is read from memory in every step)
        v4i a[kAhead];
        if constexpr (!last.value) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) a[i] = read_row<D>(k_at, i / T::kSteps, i % T::kSteps);
          next[0] = next[1] = v16f{};
        }
        float x[32], own;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          if constexpr (!last.value) {
            const int h = i / T::kSteps, j = i + kAhead;
            next[h] = mfma16<DT>(a[i % kAhead], q[i % T::kSteps], next[h]);
            if (j < kParts) a[i % kAhead] = read_row<D>(k_at, j / T::kSteps, j % T::kSteps);
          }
#pragma unroll
          for (int j = i * kEach; j < (i + 1) * kEach; ++j) x[j] = fast_exp2(__fmaf_rn(s[j / 16][j % 16], scale, minus));
#pragma unroll
          for (int j = (i - 1) * kEach; j < i * kEach; ++j)
            if (j >= 0) own = j == 0 ? x[j] : own + x[j];
          if (i > 0) pin(own);  // (added up here, not later with all of x held for it)
          if (i * kEach % 8 == 0 && i > 0) {
            const int f = i * kEach / 8 - 1;
            pr[f] = pack8<DT>(x[8 * f], x[8 * f + 1], x[8 * f + 2], x[8 * f + 3], x[8 * f + 4], x[8 * f + 5], x[8 * f + 6], x[8 * f + 7]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 32 - kEach; j < 32; ++j) own += x[j];
        sum += own;
        pr[3] = pack8<DT>(x[24], x[25], x[26], x[27], x[28], x[29], x[30], x[31]);
      }
      {
        constexpr int kParts = 4 * T::kBlocks, kEach = 16 / kParts, kAhead = 3;
        v4i a[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) a[i] = read_column<D>(v_at, i % T::kBlocks, i / T::kBlocks);
        float x = -INFINITY;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          const int j = i + kAhead;
          acc[i % T::kBlocks] = mfma16<DT>(a[i % kAhead], pr[i / T::kBlocks], acc[i % T::kBlocks]);
          if (j < kParts) a[i % kAhead] = read_column<D>(v_at, j % T::kBlocks, j / T::kBlocks);
          if constexpr (!last.value) {
#pragma unroll
            for (int l = i * kEach; l < (i + 1) * kEach; ++l) x = largest(x, next[0][l], next[1][l]);
            pin(x);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        most = x;
      }
    };
    auto step = [&](int t, v16f (&s)[2], v16f (&next)[2], auto last) {
      tile_ready<0>();
      Tile64 after64;
      if constexpr (!last.value) {
        after64.finish(p, next_lookup);
        copy_values(t + 1, next64);
        copy_keys(t + 2, after64);
        look_up(t + 3);
      }
      if (!idle) {
        compute(t, s, next, last);
        if constexpr (!last.value) hide(t + 1, next64.exist, next);
      }
      if constexpr (!last.value) {
        values_there(t + 1);
        keys_there(t + 2);
        next64 = after64;
      }
    };
    typedef std::integral_constant<bool, false> More;
    typedef std::integral_constant<bool, true> Last;
    v16f s0[2], s1[2];
    keys_there(range.from);
    tile_ready<0>();
    row_ready(q);
    copy_keys(range.from + 1, next64);
    copy_values(range.from, here64);
    if (!idle) {
      s0[0] = s0[1] = v16f{};
#pragma unroll
      for (int i = 0; i < 2 * T::kSteps; ++i)
        s0[i / T::kSteps] = mfma16<DT>(read_row<D>(k_tile(range.from) + row_at, i / T::kSteps, i % T::kSteps), q[i % T::kSteps], s0[i / T::kSteps]);
#pragma unroll
      for (int i = 0; i < 16; ++i) most = largest(most, s0[0][i], s0[1][i]);
      hide(range.from, here64.exist, s0);
    }
    keys_there(range.from + 1);
    values_there(range.from);
    int t = range.from;
#pragma unroll 1
    for (; t + 2 < range.to; t += 2) {
      step(t, s0, s1, More{});
      step(t + 1, s1, s0, More{});
    }
    if (t + 1 < range.to) {
      step(t, s0, s1, More{});
      step(t + 1, s1, s0, Last{});
    } else {
      step(t, s0, s1, Last{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may outlive the workgroup's LDS
  }
  const bool takes_part = row < e.rows, exists = row < all_rows;
  const float total = over_halves<Sum>(sum);
  if (range.runs > 1) {
    const int kept = min(all_rows, kCacheBlock);
    const int64_t at = ((int64_t)place.cut * p.runs + place.run) * kept + row - row0;
    store_column_part<D>(acc, 1.0f, p.part + at * D, hh, takes_part);
    if (takes_part && hh == 0) *reinterpret_cast<float2*>(p.part + (int64_t)p.cut * p.runs * kept * D + 2 * at) = make_float2(minus, total);
    return;
  }
  const float factor = !takes_part || total == 0.0f ? 0.0f : (p.v_scale != nullptr ? p.v_scale[hk] : 1.0f) / total;
  if (!takes_part) {
#pragma unroll
    for (int d = 0; d < T::kBlocks; ++d) acc[d] = v16f{};
  }
  const int r = min(row, all_rows - 1), l = position_of(p, r);
  store_column<DT, D>(acc, factor, p.o + b * p.o_sB + l * p.o_sL + (int64_t)(hk * p.group + r - l * p.group) * p.o_sH, hh, exists);
}

// Up to 32 query rows in all: waves share the rows and take a run's tiles in turn, each through LDS of its own, without a barrier.  A tile's values are on their way
// while its scores are formed and the next one's keys while its probabilities and their product are.  In the end the waves' sums are added up.
constexpr int kFewRows = 32, kFewWaves = 2;
// A wave's keys, values and entries.  Of 8 bits keys and values take the same place in turn, since they pass through registers: four workgroups to a
// compute unit instead of two.  (16 sequences of up to 32760 tokens, 8 heads of 128 channels: 199 us with two, 167 with four, 143, 4.4 TB/s, with the next keys and values
// asked for as soon as these are in LDS.  Without any product, exponential or write to LDS, but with the waits for LDS, it takes 131.)
template <int D, bool kEight>
constexpr int kFewWaveLds = (kEight ? 1 : 2) * Tile<D>::kBytes + 512;
template <int D, bool kEight>
constexpr int kFewLds = kFewWaves * kFewWaveLds<D, kEight>;

template <int kLater>
__device__ __forceinline__ void copies_there() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLater) : "memory");
}
// What was read of LDS is in registers: copies may go there
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void lds_copy4_from(const void* lane_at, unsigned lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(lane_at) : "memory", "m0");
#pragma clang diagnostic pop
}

template <int DT, int D, bool kEight>
__global__ __launch_bounds__(64 * kFewWaves, kEight ? 2 : 1) void sage_cache_few_kernel(const CacheAttnParams p) {
  using T = Tile<D>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, hh = lane >> 5;
  const int all_rows = p.Lq * p.group;
  const Place place = place_of(p, (int)blockIdx.x);
  const int b = place.bh / p.Hkv, hk = place.bh - b * p.Hkv;
  const Extent e = extent_of(p, b);
  const Run range = run_of(p, e, place);
  if (place.run >= range.runs) return;

  constexpr int kOwn = kFewWaveLds<D, kEight>;
  const unsigned lds = lds_base() + wave * kOwn, k_tile = lds, v_tile = lds + (kEight ? 0 : T::kBytes), entries = lds + kOwn - 512;
  const float scale = fmaxf(p.c * (p.k_scale != nullptr ? p.k_scale[hk] : 1.0f), 1.2e-38f);  // (times -infinity, where a score is hidden, still that)
  v16f acc[T::kBlocks];
#pragma unroll
  for (int d = 0; d < T::kBlocks; ++d) acc[d] = v16f{};
  float top = -INFINITY, minus = kShift<DT>, sum = 0.0f;
  const int row = m, tiles = (range.to - range.from - wave + kFewWaves - 1) / kFewWaves;  // of this wave
  auto tile_of = [&](int i) { return range.from + wave + i * kFewWaves; };
  if (range.from + wave < range.to) {
    const int32_t* table = p.pages.table + b * p.pages.sB;
    // The entries of a tile's pages, through LDS so that nothing waits for them but what is in order before them
    int slot = 0;
    auto look_up = [&](int i) {
      const int key = min(tile_of(min(i, tiles - 1)) * kTrainTile + lane, e.keys - 1), number = quotient(key, p.pages.size);
      slot = key - number * p.pages.size.by;
      lds_copy4_from(table + number, entries + (i & 1) * 256);
    };
    auto found = [&](int i, Tile64& keys) {
      const int entry = *(const __attribute__((address_space(3))) int*)(uintptr_t)(entries + (i & 1) * 256 + lane * 4);
      const bool is = (unsigned)entry < (unsigned)p.pages.pages && tile_of(i) * kTrainTile + lane < e.keys;
      keys.at = is ? (unsigned)entry * (unsigned)p.page_units + (unsigned)slot * (unsigned)p.slot_units : ~0u;
      keys.exist = __ballot(is);
    };
    using Copy = std::conditional_t<kEight, WideCopy<DT, D, 1>, PagedCopy<D, 1>>;
    constexpr int kCopies = Copy::kCopies;
    Copy k_copy(p, p.k, hk, 0, lane), v_copy(p, p.v, hk, 0, lane);
    auto copy_keys = [&](const Tile64& keys) {
      if constexpr (kEight)
        k_copy.start(p, keys, 0, lane);
      else
        k_copy.start(p, keys, k_tile, 0, lane);
    };
    auto copy_values = [&](const Tile64& keys) {
      if constexpr (kEight)
        v_copy.start(p, keys, 0, lane);
      else
        v_copy.start(p, keys, v_tile, 0, lane);
    };
    v4i q[T::kSteps];
    {
      const int r = min(row, e.rows - 1), l = position_of(p, r);
      load_row<D>(p.q + b * p.q_sB + l * p.q_sL + (int64_t)(hk * p.group + r - l * p.group) * p.q_sH, hh, p.flip, q);
    }
    Tile64 here64, next64;
    look_up(0);
    copies_there<0>();
    row_ready(q);
    found(0, here64);
    look_up(1);
    copy_keys(here64);
    copy_values(here64);
    const unsigned row_at = k_tile + row_lane_at<D>(lane), column_at = v_tile + column_lane_at<D>(lane);
    const int limit = keys_seen(p, e, row), all_see = keys_seen(p, e, 0);
    auto next_keys = [&](int i) {
      found(i + 1, next64);
      reads_done();
      look_up(i + 2);
      copy_keys(next64);
    };
    // On their way here: the entries of tile i + 1, tile i's keys, its values.  (8 bits: the next ones are asked for as soon as these are in LDS, and are there when LDS is next waited for, see
    // WideCopy: it is the compute unit's other waves that work meanwhile.)
    auto step = [&](int i, auto last) {
      copies_there<kCopies>();
      if constexpr (kEight) {
        k_copy.finish(k_tile, 0, lane);
        if constexpr (!last.value) next_keys(i);
      }
      reads_done();
      v16f s[2] = {v16f{}, v16f{}};
#pragma unroll
      for (int j = 0; j < 2 * T::kSteps; ++j)
        s[j / T::kSteps] = mfma16<DT>(read_row<D>(row_at, j / T::kSteps, j % T::kSteps), q[j % T::kSteps], s[j / T::kSteps]);
      if constexpr (!kEight && !last.value) next_keys(i);
      float most = -INFINITY;
      const int first = tile_of(i) * kTrainTile;
      if (first + kTrainTile <= all_see && here64.exist == ~UINT64_C(0)) {
#pragma unroll
        for (int j = 0; j < 16; ++j) most = largest(most, s[0][j], s[1][j]);
      } else {
        most = hide_scores(s, limit - first, here64.exist);
      }
      const float here = over_halves<Max>(most);
      if (__any(here * scale > kLazy + kShift<DT> - minus || (top == -INFINITY && here > -INFINITY))) {
        const float at = fmaxf(top, here);
        const float factor = top == -INFINITY ? 0.0f : fast_exp2((top - at) * scale);
        top = at;
        minus = at == -INFINITY ? kShift<DT> : kShift<DT> - at * scale;
        sum *= factor;
#pragma unroll
        for (int d = 0; d < T::kBlocks; ++d)
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[d][j] *= factor;
      }
      // Probabilities in two parts of 16 bits, the second what rounding takes off the first: the matrix pipes have the time while memory is waited for (64 sequences of up to
      // 8192 tokens 233.3 -> 233.9 us, one token on 32760 keys 35.1 -> 35.5), and the result's error is that of its own rounding (0.0016 for 0.0023).  Of 8 bits it costs this
      // loop 2 to 5 %, since its loads are not in flight beside the products, and the cache's own rounding is far larger: one part.
      constexpr int kParts = kEight ? 1 : 2;
      v4i pr[kParts][4];
      float own = 0.0f;  // (of the tile, as above)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = fast_exp2(__fmaf_rn(s[f / 2][8 * (f % 2) + j], scale, minus));
          own += x[j];
        }
        pr[0][f] = pack8<DT>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
        if constexpr (kParts == 2) {
          float y[8];
          widen8<DT>(make_uint4((unsigned)pr[0][f][0], (unsigned)pr[0][f][1], (unsigned)pr[0][f][2], (unsigned)pr[0][f][3]), y);
          pr[1][f] = pack8<DT>(x[0] - y[0], x[1] - y[1], x[2] - y[2], x[3] - y[3], x[4] - y[4], x[5] - y[5], x[6] - y[6], x[7] - y[7]);
        }
      }
      sum += own;
      if constexpr (last.value)
        copies_there<0>();
      else
        copies_there<kCopies + 1>();
      if constexpr (kEight) {
        v_copy.finish(v_tile, 0, lane);
        if constexpr (!last.value) copy_values(next64);
      }
      reads_done();
#pragma unroll
      for (int j = 0; j < 4 * T::kBlocks; ++j) {
        const v4i v = read_column<D>(column_at, j % T::kBlocks, j / T::kBlocks);
#pragma unroll
        for (int part = 0; part < kParts; ++part) acc[j % T::kBlocks] = mfma16<DT>(v, pr[part][j / T::kBlocks], acc[j % T::kBlocks]);
      }
      if constexpr (!last.value) {
        reads_done();
        if constexpr (!kEight) copy_values(next64);
        here64 = next64;
      }
    };
    int i = 0;
#pragma unroll 1
    for (; i + 1 < tiles; ++i) step(i, std::integral_constant<bool, false>{});
    step(i, std::integral_constant<bool, true>{});
  }
  float total = over_halves<Sum>(sum);
  // The waves' sums against one reference point (a wave whose keys are all hidden has none), added up by the first
  __syncthreads();
  typedef __attribute__((address_space(3))) float* LdsFloat;
  const LdsFloat points = (LdsFloat)(uintptr_t)(lds_base() + kFewWaves * kOwn - 512);
  const LdsFloat sums = (LdsFloat)(uintptr_t)lds_base();
  static_assert(kFewWaves == 2 && kOwn - 512 >= 64 * 4 * 16 * T::kBlocks);
  if (wave != 0) {
    if (hh == 0) {
      points[m] = minus;
      points[32 + m] = total;
    }
#pragma unroll
    for (int d = 0; d < T::kBlocks; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(16 * d + j) * 64 + lane] = acc[d][j];
  }
  __syncthreads();
  if (wave != 0) return;
  const float other_minus = points[m], other_total = points[32 + m];
  const float point = fmaxf(total != 0.0f ? -minus : -INFINITY, other_total != 0.0f ? -other_minus : -INFINITY);
  const float own_factor = total != 0.0f ? fast_exp2(-minus - point) : 0.0f, other_factor = other_total != 0.0f ? fast_exp2(-other_minus - point) : 0.0f;
#pragma unroll
  for (int d = 0; d < T::kBlocks; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[d][j] = __fmaf_rn(sums[(16 * d + j) * 64 + lane], other_factor, acc[d][j] * own_factor);
  total = __fmaf_rn(other_total, other_factor, total * own_factor);
  const bool takes_part = row < e.rows, exists = row < all_rows;
  if (range.runs > 1) {
    const int64_t at = ((int64_t)place.cut * p.runs + place.run) * all_rows + row;
    store_column_part<D>(acc, 1.0f, p.part + at * D, hh, takes_part);
    if (takes_part && hh == 0) *reinterpret_cast<float2*>(p.part + (int64_t)p.cut * p.runs * all_rows * D + 2 * at) = make_float2(-point, total);
    return;
  }
  const float factor = !takes_part || total == 0.0f ? 0.0f : (p.v_scale != nullptr ? p.v_scale[hk] : 1.0f) / total;
  if (!takes_part) {
#pragma unroll
    for (int d = 0; d < T::kBlocks; ++d) acc[d] = v16f{};
  }
  const int r = min(row, all_rows - 1), l = position_of(p, r);
  store_column<DT, D>(acc, factor, p.o + b * p.o_sB + l * p.o_sL + (int64_t)(hk * p.group + r - l * p.group) * p.o_sH, hh, exists);
}

// A row's runs joined, by a wave: each stands against a reference point of its own, which lane j holds of run j.  D / 8 lanes to a run's channels, the others have
// other runs, kEach a lane, and ask for all of them before they look at any.  Bound by latency where rows are few: 64 runs of 40 rows 4 us (one run after the other 29), 4 of
// 2048 4.8.
template <int DT, int D, int kEach>
__global__ __launch_bounds__(256) void sage_cache_join_kernel(const CacheAttnParams p) {
  constexpr int kLanes = D / 8, kSlots = 64 / kLanes;
  static_assert(kMostRuns == 64);
  const int lane = threadIdx.x & 63, part = lane % kLanes, slot = lane / kLanes, all_rows = p.Lq * p.group, kept = min(all_rows, kCacheBlock);
  const int number = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6)), at = number / kept, i = number - at * kept;
  if (at >= p.cut) return;
  Place place = block_place(p, p.whole + at);
  place.cut = at;
  const int b = place.bh / p.Hkv, hk = place.bh - b * p.Hkv, r = place.block * kCacheBlock + i;
  if (r >= all_rows) return;
  const Extent e = extent_of(p, b);
  const int runs = run_of(p, e, place).runs;
  if (runs == 1) return;
  float sum[8] = {}, total = 0.0f;
  if (r < e.rows) {
    const int64_t first = (int64_t)at * p.runs * kept + i;
    const float2 x = reinterpret_cast<const float2*>(p.part + (int64_t)p.cut * p.runs * kept * D)[first + (int64_t)min(lane, runs - 1) * kept];
    float4 lo[kEach], hi[kEach];
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const float4* values = reinterpret_cast<const float4*>(p.part + (first + (int64_t)min(slot + n * kSlots, runs - 1) * kept) * D + 8 * part);
      lo[n] = values[0];
      hi[n] = values[1];
    }
    const bool some = lane < runs && x.y != 0.0f;  // (a run whose keys are all hidden has no reference point)
    const float top = over_lanes<Max>(some ? -x.x : -INFINITY);
    const float own = some ? fast_exp2(-x.x - top) : 0.0f;
    total = over_lanes<Sum>(some ? x.y * own : 0.0f);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const float factor = __shfl(own, slot + n * kSlots);  // (of lanes without a run: 0)
      sum[0] = __fmaf_rn(lo[n].x, factor, sum[0]);
      sum[1] = __fmaf_rn(lo[n].y, factor, sum[1]);
      sum[2] = __fmaf_rn(lo[n].z, factor, sum[2]);
      sum[3] = __fmaf_rn(lo[n].w, factor, sum[3]);
      sum[4] = __fmaf_rn(hi[n].x, factor, sum[4]);
      sum[5] = __fmaf_rn(hi[n].y, factor, sum[5]);
      sum[6] = __fmaf_rn(hi[n].z, factor, sum[6]);
      sum[7] = __fmaf_rn(hi[n].w, factor, sum[7]);
    }
#pragma unroll
    for (int j = kLanes; j < 64; j <<= 1)
#pragma unroll
      for (int c = 0; c < 8; ++c) sum[c] += __shfl_xor(sum[c], j);
  }
  if (slot != 0) return;
  const int l = position_of(p, r);
  const float factor = total == 0.0f ? 0.0f : (p.v_scale != nullptr ? p.v_scale[hk] : 1.0f) / total;
  *reinterpret_cast<v4i*>(p.o + b * p.o_sB + l * p.o_sL + (int64_t)(hk * p.group + r - l * p.group) * p.o_sH + 8 * part) =
      pack8<DT>(sum[0] * factor, sum[1] * factor, sum[2] * factor, sum[3] * factor, sum[4] * factor, sum[5] * factor, sum[6] * factor, sum[7] * factor);
}

// 64 KiB of dynamic LDS and more has to be requested per kernel, once per device.
struct LdsRequest {
  std::atomic<bool> done[64];
  hipError_t make(const void* kernel, int bytes) {
    if (bytes < 65536) return hipSuccess;
    int dev = 0;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
    if (done[dev].load(std::memory_order_acquire)) return hipSuccess;
    const hipError_t f = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (f == hipSuccess) done[dev].store(true, std::memory_order_release);
    return f;
  }
};

void fill_in(CacheAttnParams& p) {
  p.group = p.Hq / p.Hkv;
  p.by_group = divisor(p.group);
  p.c = fabsf(p.sm_scale) * kLog2e;
  p.flip = p.sm_scale < 0.0f ? 0x80008000u : 0u;
  p.page_units = (int)(p.sP / 16);
  p.slot_units = (int)(p.sS / 16);
  p.blocks = (p.Lq * p.group + kCacheBlock - 1) / kCacheBlock;
  const int64_t blocks = (int64_t)p.B * p.Hkv * p.blocks, tiles = ((int64_t)p.pages.width * p.pages.size.by + kTrainTile - 1) / kTrainTile;
  const int most = (int)std::min<int64_t>(kMostRuns, (tiles + kLeastTiles - 1) / kLeastTiles);
  const double rows = std::min(p.Lq * p.group, kCacheBlock);
  p.whole = 0;
  p.cut = (int)blocks;
  p.runs = 1;
  double least = 1e30;
  if (p.Lq * p.group <= kFewRows) {
    // In us: the keys' and values' bytes at the memory's rate, half of what a wave takes for its tiles one after the other, workgroups that come and go, the second launch and
    // its bytes.  (One token on 32760 keys, 8 heads: 64 runs 28, 10 runs 52; 64 sequences of up to 8192: 2 runs 229, 4 232, 8 245; one of 2000: 17 runs 11.5, 9 12.5, 5 15.8.)
    // A compute unit has places for two workgroups of 16-bit rows of 128 channels, whose tiles fill its LDS, and for four of the others.  (64 channels with 1024 places, and with 512: 8
    // sequences of 4096 16.4 us and 18.2, 4 of 32760 58.0 and 61.7, 64 of up to 8192 127 and 131, one of 32760, 40 key heads, 72 and 75.)
    const double places = p.eight_bits || p.D == 64 ? 1024.0 : 512.0, all = 2.0 * kTrainTile * p.D * (p.eight_bits ? 1.0 / 4.2e6 : 2.0 / 5.0e6) * tiles * blocks;
    for (int n = 1; n <= most; ++n) {
      const double each = (double)((tiles + n - 1) / n), workgroups = (double)n * blocks;
      const double cost = all + 0.85 * std::ceil(each / kFewWaves) + 2.0 * std::max(1.0, workgroups / places) + (n == 1 ? 0.0 : 3.0 + 2.0 * workgroups * rows * p.D * 4.0 / 4e6);
      if (cost < 0.98 * least) {
        least = cost;
        p.runs = n;
      }
    }
    return;
  }
  // Blocks that fill whole rounds of 512 places are left whole, the others are cut so that they fill one more.  In units of a tile's time (about
  // 2 us with all there) a workgroup costs two besides its tiles, a second launch two and what its bytes take, written and read.
  constexpr int kPlaces = 512;
  constexpr double kSetup = 2.0, kJoin = 2.0, kBytesPerTile = 4e12 * 2e-6;
  p.whole = (int)(blocks / kPlaces * kPlaces);
  p.cut = (int)(blocks - p.whole);
  for (int n = 1; n <= most; ++n) {
    const double each = (double)((tiles + n - 1) / n);
    const double join = n == 1 ? 0.0 : kJoin + 2.0 * n * p.cut * 4.0 * rows * p.D / kBytesPerTile;
    const double cost = std::ceil((double)n * p.cut / kPlaces) * (each + kSetup) + join;
    if (cost < 0.97 * least) {
      least = cost;
      p.runs = n;
    }
  }
  if (p.cut == 0 || p.runs == 1) {
    p.whole = (int)blocks;
    p.cut = 0;
    p.runs = 1;
  }
}

template <int DT, int D, bool kEight>
hipError_t rows(const CacheAttnParams& p, hipStream_t s) {
  const unsigned workgroups = (unsigned)(p.whole + (int64_t)p.cut * p.runs);
  if (p.Lq * p.group <= kFewRows) {
    static LdsRequest request;
    const hipError_t e = request.make(reinterpret_cast<const void*>(&sage_cache_few_kernel<DT, D, kEight>), kFewLds<D, kEight>);
    if (e != hipSuccess) return e;
    sage_cache_few_kernel<DT, D, kEight><<<workgroups, 64 * kFewWaves, kFewLds<D, kEight>, s>>>(p);
  } else {
    constexpr int kLds = 4 * Tile<D>::kBytes;
    static LdsRequest request;
    const hipError_t e = request.make(reinterpret_cast<const void*>(&sage_cache_rows_kernel<DT, D, kEight>), kLds);
    if (e != hipSuccess) return e;
    sage_cache_rows_kernel<DT, D, kEight><<<workgroups, 256, kLds, s>>>(p);
  }
  if (p.runs > 1) {
    constexpr int kSlots = 512 / D;
    const unsigned groups = (unsigned)(((int64_t)p.cut * std::min(p.Lq * p.group, kCacheBlock) + 3) / 4);
    if (p.runs <= 2 * kSlots)
      sage_cache_join_kernel<DT, D, 2><<<groups, 256, 0, s>>>(p);
    else
      sage_cache_join_kernel<DT, D, kMostRuns / kSlots><<<groups, 256, 0, s>>>(p);
  }
  return hipGetLastError();
}
template <int DT, int D>
hipError_t of_cache(const CacheAttnParams& p, hipStream_t s) {
  return p.eight_bits ? rows<DT, D, true>(p, s) : rows<DT, D, false>(p, s);
}

}  // namespace

uint64_t cache_attn_scratch(CacheAttnParams p) {
  fill_in(p);
  if (p.runs == 1) return 0;
  return (uint64_t)p.cut * p.runs * std::min(p.Lq * p.group, kCacheBlock) * (p.D + 2) * 4;
}

hipError_t launch_cache_attn(CacheAttnParams p, void* scratch, hipStream_t s) {
  fill_in(p);
  p.part = static_cast<float*>(scratch);
  const bool bf16 = p.dtype == KSANA_SAGE_BF16;
  if (p.D == 128) return bf16 ? of_cache<KSANA_SAGE_BF16, 128>(p, s) : of_cache<KSANA_SAGE_FP16, 128>(p, s);
  return bf16 ? of_cache<KSANA_SAGE_BF16, 64>(p, s) : of_cache<KSANA_SAGE_FP16, 64>(p, s);
}

}  // namespace ksana_sage
