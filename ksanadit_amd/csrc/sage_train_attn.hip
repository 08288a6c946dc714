// Attention for training: o = softmax(c q k^T) v on 16-bit tensors with its backward pass, which recomputes the probabilities.
//
//   forward   S = c q k^T,  lse = log sum exp S,  P = exp(S - lse),  o = P v
//   backward  dv = P^T dO,  dP = dO v^T,  d = rowsum(dO o),  dS = P (dP - d),  dq = c dS k,  dk = c dS^T q
//
// Nothing of the size of S is kept: the forward pass walks the keys with a running maximum and sum, the backward pass forms S
// again from q, k and lse, once for dk and dv (a workgroup keeps keys and walks the query rows) and once for dq (it
// keeps query rows and walks the keys).  That is seven products of the backward pass where five would do with dq summed by
// atomic additions of all workgroups: their order would change the result from call to call.
//
// P and dS are rounded to the tensors' type where they become matrix operands, which have 16 bits where they are to run at this rate; S, dP, all
// sums and accumulators are fp32.  d is formed from the result as it is rounded: an unrounded one, as much memory again, leaves dq the same error
// (0.0024 in bf16), since P's roundings are in it too.
//
// Long sequences are bound by what the matrix pipes draw: with them busy 65 % (forward), 70 % (dq) and 66 % (dk and dv) of the time the
// clock falls from 2.4 to 1.7 - 1.8 GHz.  20 heads of 32760 bf16 tokens of 128 channels: forward 9.2 ms, dq 12.7, dk and dv 17.0, that
// is 1200, 1290 and 1290 TFLOP/s of the products that they form, 8 % less on slower cards (a library's product of 16384^3: 1400).  Few keys under many rows are bound by the rows' bytes
// and what a workgroup does besides its loop, 32760 rows on 512 keys, 40 heads: 422, 642 and 666 us; a few rows by a chain of latencies.
#include "sage_train_device.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace ksana_sage {

namespace {

extern __shared__ __align__(1024) char train_lds[];
__device__ __forceinline__ unsigned lds_base() { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) void*)train_lds; }

constexpr int kTrainBlock = 128;  // query rows, or keys, of a workgroup
constexpr int kMostRuns = 128;    // of a block
constexpr int kSpread = 32, kFewKeys = 128;  // keys that dq estimates a row's mean key by; blocks whose first row sees fewer than kFewKeys take the first kSpread besides
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// Rounded to fp16, probabilities relative to a row's largest would lose bits from 2^-14 on and vanish at 2^-25; scaled up as far as
// the format goes, they do so a factor of 2^6 (forward, where the reference point may lag by 2^kLazy) or 2^15 (backward) later.
constexpr float kLazy = 8.0f;
template <int DT>
constexpr float kForwardShift = DT == KSANA_SAGE_FP16 ? 6.0f : 0.0f;
template <int DT>
constexpr float kBackwardShift = DT == KSANA_SAGE_FP16 ? 15.0f : 0.0f;

struct Extent {
  int rows, keys;  // of a batch entry that take part; rows: numbered over the heads of a key head
};
__device__ __forceinline__ Extent extent_of(const TrainAttnParams& p, int b) {
  int lq = p.Lq, lk = p.Lk;
  take_counts(p.q_lens, p.k_lens, b, lq, lk);
  return Extent{lk > 0 ? lq * p.group : 0, lk};
}

// Tiles that a block of rows (of keys) walks
__device__ __forceinline__ int key_tiles_of(const TrainAttnParams& p, const Extent& e, int row0) {
  int keys = e.keys;
  if (p.causal) keys = min(keys, row_position(p, min(row0 + kTrainBlock, p.Lq * p.group) - 1) + 1);
  return row0 < e.rows ? (keys + kTrainTile - 1) / kTrainTile : 0;
}
__device__ __forceinline__ int row_tiles_of(const TrainAttnParams& p, const Extent& e, int key0, int& first) {
  const int tiles = key0 < e.keys ? (e.rows + kTrainTile - 1) / kTrainTile : 0;
  first = p.causal ? (int)min((int64_t)key0 * p.group / kTrainTile, (int64_t)tiles) : 0;
  return tiles;
}

// A lane's query row as B operands: channels 16 s + 8 hh ..
template <int D>
__device__ __forceinline__ void load_row(const uint16_t* row, int hh, uint32_t flip, v4i (&out)[Tile<D>::kSteps]) {
#pragma unroll
  for (int s = 0; s < Tile<D>::kSteps; ++s) {
    uint4 x = *reinterpret_cast<const uint4*>(row + 16 * s + 8 * hh);
    out[s] = v4i{(int)(x.x ^ flip), (int)(x.y ^ flip), (int)(x.z ^ flip), (int)(x.w ^ flip)};
  }
}

// The lane's row is here from now on.  Without this the compiler waits where its values are used, for every load under way: in a loop
// that is the next tile, in every turn.
template <int N>
__device__ __forceinline__ void row_ready(v4i (&row)[N]) {
#pragma unroll
  for (int s = 0; s < N; ++s) asm volatile("" : "+v"(row[s]));
}

// Numbers of the keys of accumulator i of 32-key block t: 32 t + 8 (i / 4) + 4 hh + i % 4
__device__ __forceinline__ constexpr int acc_row(int i) { return 8 * (i >> 2) + (i & 3); }

// ------------------------------------------------------------------------------------------------------------ forward

// A wave keeps 32 query rows (S^T = k q^T: a lane holds scores of one row) and walks tiles of 64 keys, two waves to a SIMD.  While the
// probabilities of tile t are formed and multiplied with its values, the scores of tile t + 1 are: a few vector instructions stand behind
// every matrix instruction and run beside it.  So values are wanted a step after their keys; each have two places in LDS.
// 8 heads of 16384 tokens: bf16 981 us, 1121 TFLOP/s, fp16 1030; of 64 channels 667 us, where exponentials count twice as much.  Of 128 channels 14 or 16
// registers go through memory, before the loop and behind it.
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void sage_train_fwd_kernel(const TrainAttnParams p) {
  using T = Tile<D>;
  constexpr int kWaves = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, hh = lane >> 5;
  const int all_rows = p.Lq * p.group, blocks = (all_rows + kTrainBlock - 1) / kTrainBlock;
  const TrainPlace place = train_place(p, blocks);
  const int bh = place.bh, block = blocks - 1 - place.block, b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const Extent e = extent_of(p, b);
  const int row0 = block * kTrainBlock;
  const TileRange range = run_tiles(p, place, 0, key_tiles_of(p, e, row0));
  if (place.run >= range.runs) return;

  const unsigned lds = lds_base();
  v16f acc[T::kBlocks];
#pragma unroll
  for (int d = 0; d < T::kBlocks; ++d) acc[d] = v16f{};
  float top = -INFINITY, minus = kForwardShift<DT>, sum = 0.0f;  // reference point (unscaled), what is added to scaled scores, the row's sum
  const int row = row0 + wave * 32 + m;
  if (range.from < range.to) {
    const TileCopy<D, kWaves> k_copy(p.k + b * p.ks.sB + hk * p.ks.sH, p.ks.sL, wave, lane), v_copy(p.v + b * p.vs.sB + hk * p.vs.sH, p.vs.sL, wave, lane);
    auto k_tile = [&](int t) { return lds + (t & 1) * T::kBytes; };
    auto v_tile = [&](int t) { return lds + (2 + (t & 1)) * T::kBytes; };
    auto copy_keys = [&](int t) { k_copy.start(min(t, range.to - 1) * kTrainTile, e.keys, k_tile(t), wave, lane); };
    auto copy_values = [&](int t) { v_copy.start(min(t, range.to - 1) * kTrainTile, e.keys, v_tile(t), wave, lane); };
    copy_keys(range.from);
    v4i q[T::kSteps];
    load_row<D>(p.q + b * p.qs.sB + (int64_t)hk * p.group * p.qs.sH + row_offset(p, p.qs, min(row, e.rows - 1)), hh, p.flip, q);
    const unsigned row_at = row_lane_at<D>(lane), column_at = column_lane_at<D>(lane);
    const int limit = p.causal ? min(e.keys, row_position(p, row) + 1) : e.keys;  // keys that the row sees, and that all of the wave see
    const int all_see = p.causal ? min(e.keys, row_position(p, min(row0 + wave * 32, e.rows - 1)) + 1) : e.keys;
    const bool idle = row0 + wave * 32 >= e.rows;  // a wave without rows copies its share
    float most = -INFINITY;
    auto hide = [&](int t, v16f (&s)[2]) {
      if ((t + 1) * kTrainTile <= all_see) return;
      int left = limit - t * kTrainTile - 4 * hh;
      pin(left);  // (a branch that stays one: 64 instructions for every tile otherwise)
      float x = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h][i] = 32 * h + acc_row(i) < left ? s[h][i] : -INFINITY;
        x = largest(x, s[0][i], s[1][i]);
      }
      most = x;
    };
    // Tile t: its scores in s, the largest of the lane's in `most`; forms the scores of tile t + 1 in `next` unless `last`.
    auto step = [&](int t, v16f (&s)[2], v16f (&next)[2], auto last) {
      tile_ready<0>();
      copy_values(t + 1);
      if constexpr (!last.value) copy_keys(t + 2);
      if (idle) return;
      const float here = over_halves<Max>(most);
      if (__any(here * p.c > kLazy + kForwardShift<DT> - minus || (top == -INFINITY && here > -INFINITY))) {
        const float at = fmaxf(top, here);
        const float factor = top == -INFINITY ? 0.0f : fast_exp2((top - at) * p.c);
        top = at;
        minus = at == -INFINITY ? kForwardShift<DT> : kForwardShift<DT> - at * p.c;
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
        constexpr int kParts = 2 * T::kSteps, kEach = 32 / kParts, kAhead = 3;
        v4i a[kAhead];
        if constexpr (!last.value) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) a[i] = read_row<D>(k_at, i / T::kSteps, i % T::kSteps);
          next[0] = next[1] = v16f{};
        }
        float x[32];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          if constexpr (!last.value) {
            const int h = i / T::kSteps, j = i + kAhead;
            next[h] = mfma16<DT>(a[i % kAhead], q[i % T::kSteps], next[h]);
            if (j < kParts) a[i % kAhead] = read_row<D>(k_at, j / T::kSteps, j % T::kSteps);
          }
#pragma unroll
          for (int j = i * kEach; j < (i + 1) * kEach; ++j) x[j] = fast_exp2(__fmaf_rn(s[j / 16][j % 16], p.c, minus));
#pragma unroll
          for (int j = (i - 1) * kEach; j < i * kEach; ++j)
            if (j >= 0) sum += x[j];
          pin(sum);  // (added up here, not later with all of x held for it)
          if (i * kEach % 8 == 0 && i > 0) {
            const int f = i * kEach / 8 - 1;
            pr[f] = pack8<DT>(x[8 * f], x[8 * f + 1], x[8 * f + 2], x[8 * f + 3], x[8 * f + 4], x[8 * f + 5], x[8 * f + 6], x[8 * f + 7]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 32 - kEach; j < 32; ++j) sum += x[j];
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
      if constexpr (!last.value) hide(t + 1, next);
    };
    typedef std::integral_constant<bool, false> More;
    typedef std::integral_constant<bool, true> Last;
    v16f s0[2], s1[2];
    tile_ready<0>();
    row_ready(q);
    copy_keys(range.from + 1);
    copy_values(range.from);
    if (!idle) {
      s0[0] = s0[1] = v16f{};
#pragma unroll
      for (int i = 0; i < 2 * T::kSteps; ++i)
        s0[i / T::kSteps] = mfma16<DT>(read_row<D>(k_tile(range.from) + row_at, i / T::kSteps, i % T::kSteps), q[i % T::kSteps], s0[i / T::kSteps]);
#pragma unroll
      for (int i = 0; i < 16; ++i) most = largest(most, s0[0][i], s0[1][i]);
      hide(range.from, s0);
    }
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
  const float factor = !takes_part || total == 0.0f ? 0.0f : 1.0f / total;
  const int r = min(row, all_rows - 1), l = row_position(p, r), h = hk * p.group + r - l * p.group;
  if (range.runs > 1) {
    const int64_t at = ((int64_t)place.cut * p.runs + place.run) * kTrainBlock + row - row0;
    store_column_part<D>(acc, 1.0f, p.part + at * D, hh, takes_part);
    if (takes_part && hh == 0) *reinterpret_cast<float2*>(p.part + (int64_t)p.cut * p.runs * kTrainBlock * D + 2 * at) = make_float2(minus, total);
    return;
  }
  if (!takes_part) {
#pragma unroll
    for (int d = 0; d < T::kBlocks; ++d) acc[d] = v16f{};
  }
  store_column<DT, D>(acc, factor, p.o + b * p.os.sB + l * p.os.sL + h * p.os.sH, hh, exists);
  if (exists && hh == 0 && p.lse != nullptr)
    p.lse[((int64_t)b * p.Hq + h) * p.Lq + l] = factor == 0.0f ? -INFINITY : (log2f(total) - minus) * kLn2;
}

// ------------------------------------------------------------------------------------------------------------ backward

template <int DT>
__device__ __forceinline__ float row_minus(float lse) {
  return lse == -INFINITY ? -INFINITY : kBackwardShift<DT> - lse * kLog2e;
}
constexpr int kNormRows = 64;  // rows of a workgroup (256 and a loop: 18.8 us of 40 heads of 1560 rows where this takes 10)

// Per query row -log2(e) lse (plus the shift) and -sum(dO o); in fp16 besides the largest squared norms of rows of dO and of v per block of rows.
template <int DT, int D>
__global__ __launch_bounds__(256) void sage_train_rows_kernel(const TrainAttnParams p) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;  // lanes of a row, rows at a time
  constexpr int kBlockRows = kNormRows;
  const int lane = threadIdx.x % kLanes, slot = threadIdx.x / kLanes;
  const int bh = blockIdx.y, b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const Extent e = extent_of(p, b);
  float largest = 0.0f;
  const bool of_v = (int)blockIdx.x >= p.norm_q_blocks;  // fp16 only
  if (!of_v) {
#pragma unroll
    for (int i = 0; i < kBlockRows / kRows; ++i) {
      const int r = blockIdx.x * kBlockRows + i * kRows + slot;
      float d = 0.0f, square = 0.0f;
      if (r < e.rows) {
        const int l = row_position(p, r), h = hk * p.group + r - l * p.group;
        const uint4 x = *reinterpret_cast<const uint4*>(p.d_o + b * p.dos.sB + l * p.dos.sL + h * p.dos.sH + 8 * lane);
        const uint4 y = *reinterpret_cast<const uint4*>(p.o_in + b * p.os.sB + l * p.os.sL + h * p.os.sH + 8 * lane);
        float a[8], c[8];
        widen8<DT>(x, a);
        widen8<DT>(y, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d = __fmaf_rn(a[j], c[j], d);
          square = __fmaf_rn(a[j], a[j], square);
        }
      }
#pragma unroll
      for (int j = kLanes / 2; j > 0; j >>= 1) {
        d += __shfl_xor(d, j);
        if (DT == KSANA_SAGE_FP16) square += __shfl_xor(square, j);
      }
      largest = fmaxf(largest, square);
      if (lane == 0 && r < p.row_pad) {
        float minus = -INFINITY;
        if (r < e.rows) {
          const int l = row_position(p, r), h = hk * p.group + r - l * p.group;
          const float lse = p.lse[((int64_t)b * p.Hq + h) * p.Lq + l];
          minus = row_minus<DT>(lse);
        }
        p.row_l[(int64_t)bh * p.row_pad + r] = minus;
        p.row_d[(int64_t)bh * p.row_pad + r] = -d;
      }
    }
  } else {
    const int first = ((int)blockIdx.x - p.norm_q_blocks) * kBlockRows;
#pragma unroll
    for (int i = 0; i < kBlockRows / kRows; ++i) {
      const int r = first + i * kRows + slot;
      float square = 0.0f;
      if (r < e.keys) {
        float a[8];
        widen8<DT>(*reinterpret_cast<const uint4*>(p.v + b * p.vs.sB + r * p.vs.sL + hk * p.vs.sH + 8 * lane), a);
#pragma unroll
        for (int j = 0; j < 8; ++j) square = __fmaf_rn(a[j], a[j], square);
      }
#pragma unroll
      for (int j = kLanes / 2; j > 0; j >>= 1) square += __shfl_xor(square, j);
      largest = fmaxf(largest, square);
    }
  }
  if (DT == KSANA_SAGE_FP16) {
    __shared__ float of_wave[4];
    largest = over_lanes<Max>(largest);
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = largest;
    __syncthreads();
    if (threadIdx.x == 0)
      p.norms[(int64_t)bh * p.norm_blocks + blockIdx.x] = fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
  }
}

// In fp16 dS is scaled by the power of two that brings its bound, 2 max|dO| max|v|, to one (and by 2^15 with P): gradients of any
// size, 1e-8 or 1e4, then keep the format's bits and cannot overflow it.
__device__ __forceinline__ float ds_scale(const TrainAttnParams& p, int bh, int lane) {
  const float* n = p.norms + (int64_t)bh * p.norm_blocks;
  float q = 0.0f, v = 0.0f;
  for (int i = lane; i < p.norm_blocks; i += 64) {
    const float x = n[i];
    if (i < p.norm_q_blocks)
      q = fmaxf(q, x);
    else
      v = fmaxf(v, x);
  }
  q = over_lanes<Max>(q);
  v = over_lanes<Max>(v);
  const float most = 2.0f * sqrtf(q) * sqrtf(v);
  // (not a number, infinite or zero: no scaling)
  if (!(most > 0.0f && most < INFINITY)) return 1.0f;
  int ex;
  frexpf(most, &ex);
  return ldexpf(1.0f, max(-100, min(100, -ex)));
}

// A wave keeps 32 keys and walks tiles of 64 query rows in halves: S = q k^T and dP = dO v^T (a lane holds scores of one key; dP's
// accumulators start at -d), dv^T += dO^T P, dk^T += q^T dS.  The other wave of the SIMD works beside a wave's vector instructions.
// 8 heads of 16384 tokens: bf16 1826 us, 1205 TFLOP/s, fp16 1947; of 64 channels 1011 us.
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void sage_train_dkv_kernel(const TrainAttnParams p) {
  using T = Tile<D>;
  constexpr int kWaves = 4;
  constexpr int kStage = 2 * T::kBytes + 2 * kTrainTile * 4;  // q, dO, row_l, row_d
  constexpr bool kHalf = DT == KSANA_SAGE_FP16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, hh = lane >> 5;
  const int blocks = (p.Lk + kTrainBlock - 1) / kTrainBlock;
  const TrainPlace place = train_place(p, blocks);
  const int bh = place.bh, block = place.block, b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const Extent e = extent_of(p, b);
  const int key0 = block * kTrainBlock;
  int first_tile;
  const int tiles = row_tiles_of(p, e, key0, first_tile);
  const TileRange range = run_tiles(p, place, first_tile, tiles);
  if (place.run >= range.runs) return;

  const unsigned lds = lds_base();
  v16f dk[T::kBlocks], dv[T::kBlocks];
#pragma unroll
  for (int d = 0; d < T::kBlocks; ++d) dk[d] = dv[d] = v16f{};
  float scale = 1.0f;
  const int key = key0 + wave * 32 + m;
  if (range.from < range.to) {
    const uint16_t* q_heads = p.q + b * p.qs.sB + (int64_t)hk * p.group * p.qs.sH;
    const uint16_t* do_heads = p.d_o + b * p.dos.sB + (int64_t)hk * p.group * p.dos.sH;
    const QueryCopy<D, kWaves> q_copy(p, q_heads, p.qs, lane), do_copy(p, do_heads, p.dos, lane);
    const float* row_l = p.row_l + (int64_t)bh * p.row_pad;
    const float* row_d = p.row_d + (int64_t)bh * p.row_pad;
    auto copy = [&](int t) {
      const int at = min(t, range.to - 1) * kTrainTile;
      const unsigned stage = lds + (t & 1) * kStage;
      q_copy.start(p, at, e.rows, stage, wave, lane);
      do_copy.start(p, at, e.rows, stage + T::kBytes, wave, lane);
      // (two waves each, so that every wave has as many copies in flight)
      lds_copy4_at((wave & 1 ? row_d : row_l) + at, lane * 4, stage + 2 * T::kBytes + (wave & 1) * kTrainTile * 4);
    };
    copy(range.from);
    v4i k[T::kSteps], v[T::kSteps];
    {
      const int at = min(key, e.keys - 1);
      load_row<D>(p.k + b * p.ks.sB + at * p.ks.sL + hk * p.ks.sH, hh, p.flip, k);
      load_row<D>(p.v + b * p.vs.sB + at * p.vs.sL + hk * p.vs.sH, hh, 0, v);
    }
    if constexpr (kHalf) scale = ds_scale(p, bh, lane);
    row_ready(k);
    row_ready(v);
    const unsigned row_at = row_lane_at<D>(lane), column_at = column_lane_at<D>(lane);
    const bool idle = key0 + wave * 32 >= e.keys;  // a wave without keys copies its share
    const int64_t sees_all = (int64_t)(key0 + (wave + 1) * 32 - 1) * p.group;  // the first row that sees every key of the wave
#pragma unroll 1
    for (int t = range.from; t < range.to; ++t) {
      tile_ready<0>();
      copy(t + 1);
      if (idle) continue;
      const unsigned q_tile = lds + (t & 1) * kStage, do_tile = q_tile + T::kBytes, stats = do_tile + T::kBytes;
      const bool diagonal = p.causal && (int64_t)t * kTrainTile < sees_all;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        // S, P, dv, dP, dS, dk in turn: what one part leaves is used up by the next.  The two results and the wave's keys and values take 192 of
        // 256 registers; with a half's probabilities formed behind dP's matrix instructions and dS behind those of dv, keys are
        // read back from memory: 8 % longer for 8 heads of 16384 tokens of 128 channels.  (A loop over the halves for the same reason.)
        v16f s = v16f{}, dp;
#pragma unroll
        for (int st = 0; st < T::kSteps; ++st) {
          const v4i a = read_row<D>(q_tile + row_at, h, st);
          s = mfma16<DT>(a, k[st], s);
        }
        float x[16];
        {
          v4f l[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) l[g] = *(LdsF4)(uintptr_t)(stats + (32 * h + 8 * g + 4 * hh) * 4);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = fast_exp2(__fmaf_rn(s[i], p.c, l[i >> 2][i & 3]));
        }
        if (diagonal) {
          int from = (int)min((int64_t)key * p.group - t * kTrainTile - 32 * h - 4 * hh, (int64_t)kTrainTile);
          pin(from);  // (a branch that stays one)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = acc_row(i) < from ? 0.0f : x[i];
        }
        v4i pr[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          pr[j] = pack8<DT>(x[8 * j], x[8 * j + 1], x[8 * j + 2], x[8 * j + 3], x[8 * j + 4], x[8 * j + 5], x[8 * j + 6], x[8 * j + 7]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < T::kBlocks; ++c) {
            const v4i a = read_column<D>(do_tile + column_at, c, 2 * h + j);
            dv[c] = mfma16<DT>(a, pr[j], dv[c]);
          }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v4f d = *(LdsF4)(uintptr_t)(stats + (kTrainTile + 32 * h + 8 * g + 4 * hh) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) dp[4 * g + i] = d[i];
        }
#pragma unroll
        for (int st = 0; st < T::kSteps; ++st) {
          const v4i a = read_row<D>(do_tile + row_at, h, st);
          dp = mfma16<DT>(a, v[st], dp);
        }
        __builtin_amdgcn_sched_barrier(0);  // (what the next product reads early stands in registers that are not there)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= kHalf ? dp[i] * scale : dp[i];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          pr[j] = pack8<DT>(x[8 * j], x[8 * j + 1], x[8 * j + 2], x[8 * j + 3], x[8 * j + 4], x[8 * j + 5], x[8 * j + 6], x[8 * j + 7]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < T::kBlocks; ++c) {
            const v4i a = read_column<D>(q_tile + column_at, c, 2 * h + j);
            dk[c] = mfma16<DT>(a, pr[j], dk[c]);
          }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  const float unshift = fast_exp2(-kBackwardShift<DT>);
  const bool exists = key < p.Lk;
  if (key >= e.keys) {
#pragma unroll
    for (int c = 0; c < T::kBlocks; ++c) dk[c] = dv[c] = v16f{};
  }
  if (range.runs > 1) {
    float* at = p.part + (((int64_t)place.cut * p.runs + place.run) * kTrainBlock + key - key0) * 2 * D;
    store_column_part<D>(dk, p.sm_scale * unshift / scale, at, hh, exists);
    store_column_part<D>(dv, unshift, at + D, hh, exists);
    return;
  }
  const int64_t at = (((int64_t)b * p.Lk + min(key, p.Lk - 1)) * p.Hkv + hk) * D;
  store_column<DT, D>(dk, p.sm_scale * unshift / scale, p.dk + at, hh, exists);
  store_column<DT, D>(dv, unshift, p.dv + at, hh, exists);
}

// A wave keeps 32 query rows and walks tiles of 64 keys in halves: S^T = k q^T, dP^T = v dO^T (their accumulators start at -d), dq^T +=
// k^T dS^T.  A half's vector work stands behind matrix instructions of the other half: the matrix pipes
// are busy 70 % of the time.  8 heads of 16384 tokens: bf16 1347 us, 1224 TFLOP/s, fp16 1421; of 64 channels 850 us.
//
// A row's dS sum to zero, so dq = c sum dS (k - m) for any m.  Rounded, and with d formed from the rounded result, they do not quite, and that
// carries the mean of the keys that the row attends to into dq wherever this is off zero.  The m that takes most of it away is that mean, sum P k.  It is
// estimated from kSpread keys, spread evenly over those that the block sees (where its first row sees few, from the first kSpread and as many spread over the
// others): each with its own probability, and what these leave of one shared out by the probabilities' roots, weighted with the keys that each stands for.
// (By the probabilities themselves a row of few large ones would have one key of the sample for its mean.)  As a last tile the sum of the rounded dS times their
// shares is subtracted from dS, so keys of one kind or of several, text in front of an image or a whole sequence, leave about the same error.  Relative
// error against 64 bits, bf16, 512 rows on 4352 keys N(0, 1): 0.0024, as without m.  All keys off zero by 1, 4, 8 times N(0, 1) per channel: 0.0024, without
// 0.0036, 0.012, 0.021.  The first 64, or half of them, off by 4 and not attended to: 0.0024 and 0.0025 (with the mean of the first 64 for m 0.012 in both); an
// eighth of them attended to, or half: 0.0028 and 0.0025 (without 0.011).  Rows that attend to one key or two are worse off with an estimate, 0.0034 for
// 0.0031 where scores vary by 4 and 0.0071 for 0.0058 where by 16, and a key far off that carries most of a row and is not in the sample stays as without
// (0.0073).  The mean itself, one more product, leaves 0.0019 - 0.0024 in all of these and takes a third more work.  The estimate costs 1.4 % of the pass of 32760
// rows on 512 keys; where loops have 25 tiles and more nothing shows.
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void sage_train_dq_kernel(const TrainAttnParams p) {
  using T = Tile<D>;
  constexpr int kWaves = 4;
  constexpr bool kHalf = DT == KSANA_SAGE_FP16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 31, hh = lane >> 5;
  const int all_rows = p.Lq * p.group, blocks = (all_rows + kTrainBlock - 1) / kTrainBlock;
  const TrainPlace place = train_place(p, blocks);
  const int bh = place.bh, block = blocks - 1 - place.block, b = bh / p.Hkv, hk = bh - b * p.Hkv;
  const Extent e = extent_of(p, b);
  const int row0 = block * kTrainBlock;
  const TileRange range = run_tiles(p, place, 0, key_tiles_of(p, e, row0));
  if (place.run >= range.runs) return;

  const unsigned lds = lds_base();
  v16f dq[T::kBlocks];
#pragma unroll
  for (int c = 0; c < T::kBlocks; ++c) dq[c] = v16f{};
  float scale = 1.0f;
  const int row = row0 + wave * 32 + m;
  if (!kHalf && place.run == 0 && row >= e.rows && row < p.row_pad && hh == 0) {
    p.row_l[(int64_t)bh * p.row_pad + row] = -INFINITY;
    p.row_d[(int64_t)bh * p.row_pad + row] = 0.0f;
  }
  if (range.from < range.to) {
    const TileCopy<D, kWaves> k_copy(p.k + b * p.ks.sB + hk * p.ks.sH, p.ks.sL, wave, lane), v_copy(p.v + b * p.vs.sB + hk * p.vs.sH, p.vs.sL, wave, lane);
    const int block_sees = p.causal ? min(e.keys, row_position(p, min(row0 + kTrainBlock, all_rows) - 1) + 1) : e.keys;
    const bool few = (p.causal ? min(e.keys, row_position(p, row0) + 1) : e.keys) < kFewKeys;  // that the block's first row sees
    const int spread_from = few ? kSpread : 0;
    auto copy = [&](int t) {
      const unsigned stage = lds + (t & 1) * 2 * T::kBytes;
      if (t < range.to) {
        k_copy.start(t * kTrainTile, e.keys, stage, wave, lane);
        v_copy.start(t * kTrainTile, e.keys, stage + T::kBytes, wave, lane);
      } else {
        k_copy.template start_spread<kSpread>(spread_from, block_sees, stage, wave, lane);
      }
    };
    copy(range.from);
    v4i q[T::kSteps], g[T::kSteps];
    const int r = min(row, e.rows - 1);
    load_row<D>(p.q + b * p.qs.sB + (int64_t)hk * p.group * p.qs.sH + row_offset(p, p.qs, r), hh, p.flip, q);
    load_row<D>(p.d_o + b * p.dos.sB + (int64_t)hk * p.group * p.dos.sH + row_offset(p, p.dos, r), hh, 0, g);
    float l, d;
    if constexpr (kHalf) {
      l = p.row_l[(int64_t)bh * p.row_pad + r];
      d = p.row_d[(int64_t)bh * p.row_pad + r];
      scale = ds_scale(p, bh, lane);
      l += (float)__builtin_amdgcn_frexp_expf(scale) - 1.0f;  // (a power of two: P takes dS's scale along)
    } else {
      // dO is here: what sage_train_rows_kernel would have to read it once more for is formed on the way, and kept for dk and dv
      const int at = row_position(p, r), h = hk * p.group + r - at * p.group;
      const uint16_t* o = p.o_in + b * p.os.sB + at * p.os.sL + h * p.os.sH + 8 * hh;
      const float lse = p.lse[((int64_t)b * p.Hq + h) * p.Lq + at];
      float sum[T::kSteps] = {};
#pragma unroll
      for (int s = 0; s < T::kSteps; ++s) {
        float x[8], y[8];
        widen8<DT>(*reinterpret_cast<const uint4*>(o + 16 * s), x);
        widen8<DT>(__builtin_bit_cast(uint4, g[s]), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[s] = __fmaf_rn(x[j], y[j], sum[s]);
      }
      // (added up in the order of that kernel's lanes: dk and dv have the same bits whether dq is wanted or not)
#pragma unroll
      for (int n = T::kSteps / 2; n > 0; n /= 2)
#pragma unroll
        for (int s = 0; s < n; ++s) sum[s] += sum[s + n];
      l = row_minus<DT>(lse);
      d = -over_halves<Sum>(sum[0]);
      if (place.run == 0 && hh == 0 && row < e.rows) {
        p.row_l[(int64_t)bh * p.row_pad + row] = l;
        p.row_d[(int64_t)bh * p.row_pad + row] = d;
      }
    }
    float sum_ds = 0.0f;
    row_ready(q);
    row_ready(g);
    const unsigned row_at = row_lane_at<D>(lane), column_at = column_lane_at<D>(lane);
    const int limit = p.causal ? min(e.keys, row_position(p, row) + 1) : e.keys;
    const int all_see = p.causal ? min(e.keys, row_position(p, min(row0 + wave * 32, e.rows - 1)) + 1) : e.keys;
    const bool idle = row0 + wave * 32 >= e.rows;  // a wave without rows copies its share
    // A step of the tile: an operand read ahead, a matrix instruction, and vector work of a part of the 16 elements of a half
    constexpr int kSteps = T::kSteps, kEach = 16 / kSteps, kAhead = 3;
    v16f s[2], dp[2];
    v4i ds[2][2], a[kAhead];
    auto rows_product = [&](unsigned rows, int h, const v4i(&other)[kSteps], v16f& to, auto&& beside) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) a[i] = read_row<D>(rows, h, i);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        to = mfma16<DT>(a[i % kAhead], other[i], to);
        if (i + kAhead < kSteps) a[i % kAhead] = read_row<D>(rows, h, i + kAhead);
        beside(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto columns_product = [&](unsigned columns, int h, auto&& beside) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) a[i] = read_column<D>(columns, i % T::kBlocks, 2 * h + i / T::kBlocks);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int j = i + kAhead;
        dq[i % T::kBlocks] = mfma16<DT>(a[i % kAhead], ds[h][i / T::kBlocks], dq[i % T::kBlocks]);
        if (j < kSteps) a[i % kAhead] = read_column<D>(columns, j % T::kBlocks, 2 * h + j / T::kBlocks);
        beside(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto pack = [&](int h, int f) {
      return pack8<DT>(s[h][8 * f], s[h][8 * f + 1], s[h][8 * f + 2], s[h][8 * f + 3], s[h][8 * f + 4], s[h][8 * f + 5], s[h][8 * f + 6], s[h][8 * f + 7]);
    };
    auto nothing = [](int) {};
#pragma unroll 1
    for (int t = range.from; t < range.to; ++t) {
      tile_ready<0>();
      copy(t + 1);
      if (idle) continue;
      unsigned k_rows = lds + (t & 1) * 2 * T::kBytes + row_at, v_rows = k_rows + T::kBytes, k_columns = lds + (t & 1) * 2 * T::kBytes + column_at;
      pin(k_rows);  // (one address and constants each)
      pin(v_rows);
      pin(k_columns);
      auto probabilities = [&](int h) {
        return [&, h](int i) {
#pragma unroll
          for (int j = i * kEach; j < (i + 1) * kEach; ++j) s[h][j] = fast_exp2(__fmaf_rn(s[h][j], p.c, l));
        };
      };
      auto gradients = [&](int h) {
        return [&, h](int i) {
#pragma unroll
          for (int j = i * kEach; j < (i + 1) * kEach; ++j) s[h][j] *= dp[h][j];
          if ((i + 1) * kEach % 8 == 0) {
            const int f = (i + 1) * kEach / 8 - 1;
            ds[h][f] = pack(h, f);
            sum_ds = add8<DT>(ds[h][f], sum_ds);
          }
        };
      };
      auto hide = [&](int h) {
        if ((t + 1) * kTrainTile <= all_see) return;
        int left = limit - t * kTrainTile - 32 * h - 4 * hh;
        pin(left);  // (a branch that stays one)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] = acc_row(i) < left ? s[h][i] : 0.0f;
      };
      s[0] = s[1] = v16f{};
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[0][i] = dp[1][i] = d;
      rows_product(k_rows, 0, q, s[0], nothing);
      rows_product(v_rows, 0, g, dp[0], probabilities(0));
      hide(0);
      rows_product(k_rows, 1, q, s[1], gradients(0));
      rows_product(v_rows, 1, g, dp[1], probabilities(1));
      hide(1);
      columns_product(k_columns, 0, gradients(1));
      columns_product(k_columns, 1, nothing);
    }
    tile_ready<0>();  // (and no copy outlives the workgroup's LDS)
    if (!idle) {
      const unsigned tile = lds + (range.to & 1) * 2 * T::kBytes;
      float most = -INFINITY, total = 0.0f;
      auto scores = [&](int h, int left) {  // of the half's first `left` keys
        s[h] = v16f{};
        rows_product(tile + row_at, h, q, s[h], nothing);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[h][i] = acc_row(i) < left - 4 * hh ? s[h][i] : -INFINITY;
          most = fmaxf(most, s[h][i]);
        }
      };
      const int spread = block_sees - spread_from, seen = limit - spread_from;  // key j of the first half is key j spread / kSpread of those
      scores(0, spread >= kSpread ? (kSpread * seen + spread - 1) / spread : seen);
      if (few) scores(1, limit);
      most = fmaxf(over_halves<Max>(most) * p.c, -3e38f);  // (scores that are all out of fp32's range: no shares)
      // roots of the probabilities relative to the largest: their sum, and what the keys have of the row
      float mass = 0.0f;
      auto roots = [&](int h, float weight) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[h][i] = fast_exp2(0.5f * __fmaf_rn(s[h][i], p.c, -most));
          total = __fmaf_rn(s[h][i], weight, total);
          mass = __fmaf_rn(s[h][i], s[h][i], mass);
        }
      };
      const float weight = fmaxf(1.0f, (float)spread / kSpread);  // (one key for so many)
      roots(0, weight);
      if (few) roots(1, 1.0f);
      total = over_halves<Sum>(total);
      sum_ds = -over_halves<Sum>(sum_ds);
      const float minus = kHalf ? l - kBackwardShift<DT> - ((float)__builtin_amdgcn_frexp_expf(scale) - 1.0f) : l;  // -log2(e) lse
      const float largest_one = fast_exp2(most + minus), rest = fmaxf(0.0f, 1.0f - over_halves<Sum>(mass) * largest_one);
      const float own = sum_ds * largest_one, share = total > 0.0f ? sum_ds * rest / total : 0.0f;  // (not a number: nor is the row's dq)
      auto subtract = [&](int h, float weight) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] *= __fmaf_rn(s[h][i], own, weight * share);
#pragma unroll
        for (int f = 0; f < 2; ++f) ds[h][f] = pack(h, f);
        columns_product(tile + column_at, h, nothing);
        if (range.runs == 1) return;
        // a run's dS sum to more than roundings: what is left of the shares when they are rounded counts too
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          float x[8];
          widen8<DT>(__builtin_bit_cast(uint4, ds[h][f]), x);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[h][8 * f + j] -= x[j];
          ds[h][f] = pack(h, f);
        }
        columns_product(tile + column_at, h, nothing);
      };
      subtract(0, weight);
      if (few) subtract(1, 1.0f);
    }
  }
  const float unshift = fast_exp2(-kBackwardShift<DT>);
  const bool exists = row < all_rows;
  const int r = min(row, all_rows - 1), at = row_position(p, r), h = hk * p.group + r - at * p.group;
  if (row >= e.rows) {
#pragma unroll
    for (int c = 0; c < T::kBlocks; ++c) dq[c] = v16f{};
  }
  if (range.runs > 1) {
    store_column_part<D>(dq, p.sm_scale * unshift / scale, p.part + (((int64_t)place.cut * p.runs + place.run) * kTrainBlock + row - row0) * D, hh, exists);
    return;
  }
  store_column<DT, D>(dq, p.sm_scale * unshift / scale, p.dq + (((int64_t)b * p.Lq + at) * p.Hq + h) * D, hh, exists);
}

// ------------------------------------------------------------------------------------------------------------ runs joined

// Bound by the bytes of the runs and, of few rows, by latency.  Eight channels per lane; kSlots groups of lanes share a row's runs and
// add their sums up in a fixed order (many runs of few rows; 64 runs of one row, 40 heads: 4 us).
template <int kSlots>
__device__ __forceinline__ void add_slots(float (&x)[9], int slot, int lanes, int lane) {
  if constexpr (kSlots > 1) {
    __shared__ float all[256 * 9];
#pragma unroll
    for (int i = 0; i < 9; ++i) all[i * 256 + threadIdx.x] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      float sum = 0.0f;
      for (int j = 0; j < kSlots; ++j) sum += all[i * 256 + j * lanes + lane];
      x[i] = sum;
    }
  }
}

// A run's sums stand against a reference point of its own.  With slots a row has a workgroup, which asks for all it reads before it looks at any
// of it (reference points one load after the other, then sums: 6.3 us for the 64 runs of a row of 40 heads, this 4).
template <int DT, int D, int kSlots>
__global__ __launch_bounds__(256) void sage_train_join_fwd_kernel(const TrainAttnParams p, const int groups) {
  constexpr int kLanes = D / 8, kRows = 256 / (kLanes * kSlots);
  const int lane = threadIdx.x % kLanes, slot = kSlots > 1 ? threadIdx.x / kLanes : 0, own = kSlots > 1 ? 0 : threadIdx.x / kLanes;
  static_assert(kSlots == 1 || kRows == 1);
  const int all_rows = p.Lq * p.group, blocks = (all_rows + kTrainBlock - 1) / kTrainBlock;
  TrainPlace place = block_place(p, blocks, p.whole + (int)blockIdx.x / groups);
  place.cut = (int)blockIdx.x / groups;
  const int bh = place.bh, b = bh / p.Hkv, hk = bh - b * p.Hkv, row0 = (blocks - 1 - place.block) * kTrainBlock;
  const int i = (int)blockIdx.x % groups * kRows + own, r = row0 + i;
  const Extent e = extent_of(p, b);
  const int runs = run_tiles(p, place, 0, key_tiles_of(p, e, row0)).runs;
  if (runs == 1 || r >= all_rows) return;  // (with slots, of the whole workgroup)
  const int64_t first = (int64_t)place.cut * p.runs * kTrainBlock + i;
  const float2* ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.cut * p.runs * kTrainBlock * D);
  auto point = [&](int j) { return ml[first + (int64_t)j * kTrainBlock]; };
  auto values = [&](int j) { return reinterpret_cast<const float4*>(p.part + (first + (int64_t)j * kTrainBlock) * D + 8 * lane); };
  float sum[9] = {}, top = -INFINITY;
  auto add = [&](const float4& lo, const float4& hi, float factor) {
    sum[0] = __fmaf_rn(lo.x, factor, sum[0]);
    sum[1] = __fmaf_rn(lo.y, factor, sum[1]);
    sum[2] = __fmaf_rn(lo.z, factor, sum[2]);
    sum[3] = __fmaf_rn(lo.w, factor, sum[3]);
    sum[4] = __fmaf_rn(hi.x, factor, sum[4]);
    sum[5] = __fmaf_rn(hi.y, factor, sum[5]);
    sum[6] = __fmaf_rn(hi.z, factor, sum[6]);
    sum[7] = __fmaf_rn(hi.w, factor, sum[7]);
  };
  if constexpr (kSlots > 1) {
    constexpr int kOwn = (kMostRuns + kSlots - 1) / kSlots;
    static_assert(kMostRuns <= 256);
    __shared__ float factors[kMostRuns], of_wave[2][4];
    if (r < e.rows) {  // (the whole workgroup)
      const int j = threadIdx.x;
      const float2 x = j < runs ? point(j) : make_float2(0.0f, 0.0f);
      float4 lo[kOwn], hi[kOwn];
#pragma unroll
      for (int n = 0; n < kOwn; ++n) {
        const float4* o = values(min(slot + n * kSlots, runs - 1));
        lo[n] = o[0];
        hi[n] = o[1];
      }
      const float most = over_lanes<Max>(x.y != 0.0f ? -x.x : -INFINITY);  // (a run whose keys are all hidden has no reference point)
      if ((j & 63) == 0) of_wave[0][j >> 6] = most;
      __syncthreads();
      top = fmaxf(fmaxf(of_wave[0][0], of_wave[0][1]), fmaxf(of_wave[0][2], of_wave[0][3]));
      const float factor = x.y != 0.0f ? fast_exp2(-x.x - top) : 0.0f;
      if (j < kMostRuns) factors[j] = factor;
      const float total = over_lanes<Sum>(x.y * factor);
      if ((j & 63) == 0) of_wave[1][j >> 6] = total;
      __syncthreads();
#pragma unroll
      for (int n = 0; n < kOwn; ++n)
        if (slot + n * kSlots < runs) add(lo[n], hi[n], factors[slot + n * kSlots]);
    }
    add_slots<kSlots>(sum, slot, kLanes, lane);
    if (slot != 0) return;
    sum[8] = r < e.rows ? of_wave[1][0] + of_wave[1][1] + of_wave[1][2] + of_wave[1][3] : 0.0f;
  } else if (r < e.rows) {
    for (int j = lane; j < runs; j += kLanes) {
      const float2 x = point(j);
      top = x.y != 0.0f ? fmaxf(top, -x.x) : top;
    }
#pragma unroll
    for (int j = kLanes / 2; j > 0; j >>= 1) top = fmaxf(top, __shfl_xor(top, j));
#pragma unroll 4
    for (int j = 0; j < runs; ++j) {
      const float2 x = point(j);
      const float factor = x.y != 0.0f ? fast_exp2(-x.x - top) : 0.0f;
      sum[8] = __fmaf_rn(x.y, factor, sum[8]);
      add(values(j)[0], values(j)[1], factor);
    }
  }
  const int l = row_position(p, r), h = hk * p.group + r - l * p.group;
  const float factor = sum[8] == 0.0f ? 0.0f : 1.0f / sum[8];
  *reinterpret_cast<v4i*>(p.o + b * p.os.sB + l * p.os.sL + h * p.os.sH + 8 * lane) =
      pack8<DT>(sum[0] * factor, sum[1] * factor, sum[2] * factor, sum[3] * factor, sum[4] * factor, sum[5] * factor, sum[6] * factor, sum[7] * factor);
  if (lane == 0 && p.lse != nullptr) p.lse[((int64_t)b * p.Hq + h) * p.Lq + l] = sum[8] == 0.0f ? -INFINITY : (log2f(sum[8]) + top) * kLn2;
}

// Sums of the runs' gradients: of query rows (kKeys false) or of keys, whose two gradients lie side by side
template <int DT, int D, bool kKeys, int kSlots>
__global__ __launch_bounds__(256) void sage_train_join_bwd_kernel(const TrainAttnParams p, const int groups) {
  constexpr int kWidth = kKeys ? 2 * D : D, kLanes = kWidth / 8, kRows = kSlots > 1 ? 1 : 256 / kLanes;
  static_assert(kSlots == 1 || kLanes * kSlots == 256);
  const int lane = threadIdx.x % kLanes, slot = kSlots > 1 ? threadIdx.x / kLanes : 0, own = kSlots > 1 ? 0 : threadIdx.x / kLanes;
  const int all = kKeys ? p.Lk : p.Lq * p.group, blocks = (all + kTrainBlock - 1) / kTrainBlock;
  TrainPlace place = block_place(p, blocks, p.whole + (int)blockIdx.x / groups);
  place.cut = (int)blockIdx.x / groups;
  const int bh = place.bh, b = bh / p.Hkv, hk = bh - b * p.Hkv, row0 = (kKeys ? place.block : blocks - 1 - place.block) * kTrainBlock;
  const int i = (int)blockIdx.x % groups * kRows + own, r = row0 + i;
  const Extent e = extent_of(p, b);
  int from = 0;
  const int to = kKeys ? row_tiles_of(p, e, row0, from) : key_tiles_of(p, e, row0);
  const int runs = run_tiles(p, place, from, to).runs;
  if (runs == 1 || r >= all) return;
  const int64_t first = (int64_t)place.cut * p.runs * kTrainBlock + i;
  float sum[9] = {};
#pragma unroll 4
  for (int j = slot; j < runs; j += kSlots) {
    const float4* x = reinterpret_cast<const float4*>(p.part + (first + (int64_t)j * kTrainBlock) * kWidth + 8 * lane);
    const float4 lo = x[0], hi = x[1];
    sum[0] += lo.x;
    sum[1] += lo.y;
    sum[2] += lo.z;
    sum[3] += lo.w;
    sum[4] += hi.x;
    sum[5] += hi.y;
    sum[6] += hi.z;
    sum[7] += hi.w;
  }
  add_slots<kSlots>(sum, slot, kLanes, lane);
  if (slot != 0) return;
  uint16_t* out;
  if constexpr (kKeys) {
    out = (8 * lane < D ? p.dk : p.dv) + (((int64_t)b * p.Lk + r) * p.Hkv + hk) * D + 8 * lane % D;
  } else {
    const int l = row_position(p, r);
    out = p.dq + (((int64_t)b * p.Lq + l) * p.Hq + hk * p.group + r - l * p.group) * D + 8 * lane;
  }
  *reinterpret_cast<v4i*>(out) = pack8<DT>(sum[0], sum[1], sum[2], sum[3], sum[4], sum[5], sum[6], sum[7]);
}

// ------------------------------------------------------------------------------------------------------------ launches

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

void fill_in(TrainAttnParams& p) {
  p.group = p.Hq / p.Hkv;
  p.group_inv = (unsigned)((UINT64_C(0x100000000) + p.group - 1) / p.group);
  p.group_shift = p.group <= 16 && (p.group & (p.group - 1)) == 0 ? __builtin_ctz((unsigned)p.group) : -1;
  p.c = std::max(fabsf(p.sm_scale) * kLog2e, 1.2e-38f);  // (times -infinity, where a score is hidden, still that)
  p.flip = p.sm_scale < 0.0f ? 0x80008000u : 0u;
  p.row_pad = (p.Lq * p.group + kTrainTile - 1) / kTrainTile * kTrainTile;
  p.norm_q_blocks = (p.row_pad + kNormRows - 1) / kNormRows;
  p.norm_blocks = p.norm_q_blocks + (p.dtype == KSANA_SAGE_FP16 ? (p.Lk + kNormRows - 1) / kNormRows : 0);
}

// How a launch of `blocks` blocks that walk at most `tiles` tiles each is cut, with `bytes` of results to a block.  `places`: two
// workgroups to each of 256 compute units, three of dk and dv of 64 channels (12 heads of 4096 tokens: 113 + 11 us, counted as two 142).
// In units of a tile's time (about 2 us with all there), a workgroup costs kSetup besides its tiles, a launch that joins runs kJoin and
// what its bytes take, written and read.  Blocks that cost the same: as many as fill whole rounds are
// left whole, the others are cut so that they fill one more.  Others (`differ`; of a causal call's tiles half are there): all whole or all in
// runs of one length.  Whole ones come with the longest first, so that the short ones fill up what those leave of the last round, unless
// there are so few that two long ones share a place; runs need whole rounds, or half a run's time besides their mean.  (16 heads of 8192
// causal tokens: rows whole 276 + 372 us, forward and dq (without what it does about m), in two runs 291 + 387 and 34 for the joins; on 4 key heads, dk and dv: keys whole
// 1120, in 3 runs 594 + 12, in 5 618 + 17, in 7 587 + 21.)
struct TrainCut {
  int whole, cut, runs, run_tiles;
  uint64_t part(int width) const { return runs > 1 ? (uint64_t)cut * runs * kTrainBlock * width * 4 : 0; }
};
TrainCut cut_of(int64_t blocks, int tiles, double bytes, bool differ, double share, int places) {
  constexpr double kSetup = 2.0, kJoin = 2.0, kBytesPerTile = 4e12 * 2e-6;
  const int whole = differ ? 0 : (int)(blocks / places * places);
  const int64_t rest = blocks - whole;
  double least = 1e30;
  int best = tiles;  // of a run
  // a launch holds fewer than 2^24 workgroups, and a join has up to 16 of them to a block
  const int most = rest > (1 << 19) ? 1 : (int)std::min<int64_t>(std::min(tiles, kMostRuns), ((1 << 24) - 1 - whole) / std::max<int64_t>(rest, 1));
  for (int n = 1; n <= most; ++n) {
    const int each = (tiles + n - 1) / n;
    const double join = n == 1 ? 0.0 : kJoin + 2.0 * n * rest * bytes * share / kBytesPerTile;
    const double number = rest * (share < 1.0 && n > 1 ? share * tiles / each + 0.5 : (double)((tiles + each - 1) / each));  // of runs that are there
    double cost = std::ceil(number / places) * (each + kSetup);
    if (differ && n == 1 && share < 1.0) {
      cost = std::max(tiles + kSetup, rest * (share * tiles + kSetup) / places);
      // (the (i places + 1)-th longest block is one of i + 1 in its place)
      for (int i = 1; i < 8 && (int64_t)i * places < rest; ++i) cost = std::max(cost, (i + 1) * (tiles * (1.0 - (double)i * places / rest) + kSetup));
    } else if (differ) {
      cost = std::min(cost, std::max(number * (each + kSetup) / places + 0.5 * each, each + kSetup));
    }
    cost += join;
    if (cost < 0.97 * least) {
      least = cost;
      best = each;
    }
  }
  const int runs = (tiles + best - 1) / best;
  if (runs == 1 && !differ) return TrainCut{(int)(blocks / 8 * 8), (int)(blocks % 8), 1, tiles};
  return TrainCut{whole, (int)rest, runs, best};
}
struct TrainCuts {
  TrainCut fwd, dkv, dq;
};
TrainCuts train_cuts(const TrainAttnParams& p) {
  const int64_t heads = (int64_t)p.B * p.Hkv, rows = (int64_t)p.Lq * p.group;
  const int64_t row_blocks = heads * ((rows + kTrainBlock - 1) / kTrainBlock), key_blocks = heads * ((p.Lk + kTrainBlock - 1) / kTrainBlock);
  const int key_tiles = ((p.causal ? std::min(p.Lk, p.Lq) : p.Lk) + kTrainTile - 1) / kTrainTile, row_tiles = (int)((rows + kTrainTile - 1) / kTrainTile);
  const bool differ = p.causal || p.q_lens != nullptr || p.k_lens != nullptr;
  const double share = p.causal && p.Lq > 1 ? 0.5 : 1.0, row_bytes = 4.0 * std::min<int64_t>(rows, kTrainBlock) * p.D;
  const TrainCut of_rows = cut_of(row_blocks, key_tiles, row_bytes, differ, share, 512);
  return TrainCuts{of_rows, cut_of(key_blocks, row_tiles, 8.0 * std::min(p.Lk, kTrainBlock) * p.D, differ, share, p.D == 64 ? 768 : 512), of_rows};
}
void take_cut(TrainAttnParams& p, const TrainCut& c) {
  p.whole = c.whole;
  p.cut = c.cut;
  p.runs = c.runs;
  p.run_tiles = c.run_tiles;
}
unsigned workgroups(const TrainAttnParams& p) { return (unsigned)(p.whole + (int64_t)p.cut * p.runs); }
// Rows of a block that the joins look at
int joined_rows(int64_t all) { return (int)std::min<int64_t>(all, kTrainBlock); }
// Many runs of few rows (of all blocks): lanes share a row's.  Forward and dq, 64 runs of 40 rows: 4 and 4 us, one lane after the other 20 and more; 22 of
// 960 rows: 7.3 and 7.3, 8.9 and 10.8; 16 of 4096: 15.8 and 11.2, 7.3 and 6.6; 24 of 1200 rows of 64 channels: 15.8 and 13.0, 5.4 and 5.6.
constexpr int kManyRuns = 16, kFewJoined = 1024;

template <int DT, int D>
hipError_t fwd(TrainAttnParams p, hipStream_t s) {
  constexpr int kLds = 4 * Tile<D>::kBytes;
  static LdsRequest request;
  const hipError_t e = request.make(reinterpret_cast<const void*>(&sage_train_fwd_kernel<DT, D>), kLds);
  if (e != hipSuccess) return e;
  sage_train_fwd_kernel<DT, D><<<workgroups(p), 256, kLds, s>>>(p);
  if (p.runs > 1) {
    constexpr int kLanes = D / 8;
    const int rows = joined_rows((int64_t)p.Lq * p.group), groups = (rows * kLanes + 255) / 256;  // workgroups of a block
    if (p.runs >= kManyRuns && (int64_t)rows * p.cut <= kFewJoined)
      sage_train_join_fwd_kernel<DT, D, 256 / kLanes><<<(unsigned)((int64_t)rows * p.cut), 256, 0, s>>>(p, rows);
    else
      sage_train_join_fwd_kernel<DT, D, 1><<<(unsigned)((int64_t)groups * p.cut), 256, 0, s>>>(p, groups);
  }
  return hipGetLastError();
}

template <int DT, int D, bool kKeys>
void join_bwd(const TrainAttnParams& p, int64_t all, hipStream_t s) {
  if (p.runs == 1) return;
  constexpr int kLanes = (kKeys ? 2 : 1) * D / 8;
  const int rows = joined_rows(all), groups = (rows * kLanes + 255) / 256;
  if (p.runs >= kManyRuns && (int64_t)rows * p.cut <= kFewJoined)
    sage_train_join_bwd_kernel<DT, D, kKeys, 256 / kLanes><<<(unsigned)((int64_t)rows * p.cut), 256, 0, s>>>(p, rows);
  else
    sage_train_join_bwd_kernel<DT, D, kKeys, 1><<<(unsigned)((int64_t)groups * p.cut), 256, 0, s>>>(p, groups);
}

template <int DT, int D>
hipError_t bwd(TrainAttnParams p, const TrainCuts& cuts, hipStream_t s) {
  hipError_t e = hipSuccess;
  // in bf16 the rows' numbers come along with dq, where that is wanted
  if (DT == KSANA_SAGE_FP16 || p.dq == nullptr) {
    sage_train_rows_kernel<DT, D><<<dim3(p.norm_blocks, p.B * p.Hkv), 256, 0, s>>>(p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.dq != nullptr) {
    constexpr int kLds = 2 * 2 * Tile<D>::kBytes;
    static LdsRequest request;
    e = request.make(reinterpret_cast<const void*>(&sage_train_dq_kernel<DT, D>), kLds);
    if (e != hipSuccess) return e;
    take_cut(p, cuts.dq);
    sage_train_dq_kernel<DT, D><<<workgroups(p), 256, kLds, s>>>(p);
    join_bwd<DT, D, false>(p, (int64_t)p.Lq * p.group, s);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.dk == nullptr) return hipSuccess;
  constexpr int kLds = 2 * (2 * Tile<D>::kBytes + 2 * kTrainTile * 4);
  static LdsRequest request;
  e = request.make(reinterpret_cast<const void*>(&sage_train_dkv_kernel<DT, D>), kLds);
  if (e != hipSuccess) return e;
  take_cut(p, cuts.dkv);
  sage_train_dkv_kernel<DT, D><<<workgroups(p), 256, kLds, s>>>(p);
  join_bwd<DT, D, true>(p, p.Lk, s);
  return hipGetLastError();
}

uint64_t up256(uint64_t x) { return (x + 255) & ~UINT64_C(255); }

}  // namespace

TrainAttnScratch train_attn_scratch(const TrainAttnParams& call, bool backward) {
  TrainAttnParams p = call;
  fill_in(p);
  const TrainCuts cuts = train_cuts(p);
  TrainAttnScratch out{};
  if (!backward) {
    out.bytes = up256(cuts.fwd.part(p.D + 2));
    return out;
  }
  const uint64_t heads = (uint64_t)p.B * p.Hkv, rows = up256(heads * p.row_pad * 4);
  out.row_l = 0;
  out.row_d = rows;
  out.norms = 2 * rows;
  out.part = out.norms + up256(heads * p.norm_blocks * 4);
  out.bytes = out.part + up256(std::max(cuts.dkv.part(2 * p.D), cuts.dq.part(p.D)));  // (one after the other)
  return out;
}

hipError_t launch_train_attn_fwd(TrainAttnParams p, void* scratch, hipStream_t s) {
  fill_in(p);
  take_cut(p, train_cuts(p).fwd);
  p.part = static_cast<float*>(scratch);
  const bool bf16 = p.dtype == KSANA_SAGE_BF16;
  if (p.D == 128) return bf16 ? fwd<KSANA_SAGE_BF16, 128>(p, s) : fwd<KSANA_SAGE_FP16, 128>(p, s);
  return bf16 ? fwd<KSANA_SAGE_BF16, 64>(p, s) : fwd<KSANA_SAGE_FP16, 64>(p, s);
}

hipError_t launch_train_attn_bwd(TrainAttnParams p, void* scratch, hipStream_t s) {
  const TrainAttnScratch at = train_attn_scratch(p, true);
  fill_in(p);
  const TrainCuts cuts = train_cuts(p);
  char* base = static_cast<char*>(scratch);
  p.row_l = reinterpret_cast<float*>(base + at.row_l);
  p.row_d = reinterpret_cast<float*>(base + at.row_d);
  p.norms = reinterpret_cast<float*>(base + at.norms);
  p.part = reinterpret_cast<float*>(base + at.part);
  const bool bf16 = p.dtype == KSANA_SAGE_BF16;
  if (p.D == 128) return bf16 ? bwd<KSANA_SAGE_BF16, 128>(p, cuts, s) : bwd<KSANA_SAGE_FP16, 128>(p, cuts, s);
  return bf16 ? bwd<KSANA_SAGE_BF16, 64>(p, cuts, s) : bwd<KSANA_SAGE_FP16, 64>(p, cuts, s);
}

}  // namespace ksana_sage
