// What the kernels of the training attention share: operand types, tiles of 16-bit rows in LDS and the ways they are read.
//
// Matrix instruction: D = A B + C of 32 x 32 with 16 products per element.  Lane l (column or row m = l % 32, hh = l / 32) holds
// eight values of A's row m and of B's column m, numbers 8 hh + j, and sixteen of C and D: column m, rows 8 (i / 4) + 4 hh + i % 4.
// Products of a sum may come in any order as long as A and B agree.  So the accumulators of one product, packed to 16 bits, are
// the B operand of the next one without leaving their lane: value j of step t of a lane is row 16 t + 8 (j / 4) + 4 hh + j % 4, and
// A's rows, which lie across the memory rows there, are read from LDS with the transposing read in that order.
#pragma once

#include "sage_attn_device.h"
#include "sage_kernels.h"
#include "sage_train.h"

namespace ksana_sage {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

constexpr int kTrainTile = 64;  // rows of a tile in LDS: keys, or query rows

template <int DT>
__device__ __forceinline__ v16f mfma16(const v4i& a, const v4i& b, const v16f& c) {
  if constexpr (DT == KSANA_SAGE_BF16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
}

// Eight fp32 values rounded to nearest, in operand order
template <int DT>
__device__ __forceinline__ v4i pack8(float a, float b, float c, float d, float e, float f, float g, float h) {
  const uint2 lo = half4<DT>(a, b, c, d), hi = half4<DT>(e, f, g, h);
  return v4i{(int)lo.x, (int)lo.y, (int)hi.x, (int)hi.y};
}

// sum + the eight values of an operand, as they are rounded
template <int DT>
__device__ __forceinline__ float add8(const v4i& x, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pair = x[i];  // (a vector's element is no operand of a bit cast: the first is taken)
    if constexpr (DT == KSANA_SAGE_BF16) {
      typedef __bf16 v2 __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, pair), __builtin_bit_cast(v2, 0x3f803f80), sum, false);
    } else {
      typedef _Float16 v2 __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, pair), __builtin_bit_cast(v2, 0x3c003c00), sum, false);
    }
  }
  return sum;
}

// A tile: 64 rows of D 16-bit channels.  A copy instruction of a wave fills 1 KiB in a row with 64 pieces of 16 bytes: whole rows, that
// are not neighbours.  Which rows share a copy and how far apart the copies lie is chosen so that row r starts 64 (r % 4) + 16 (r / 4 % 4)
// bytes into the 256 that the banks hold side by side: sixteen lanes that read one piece of sixteen rows, and 32 lanes that read 64 bytes
// of four rows (the transposing read), then meet in no bank, and every read of a lane is one address and a constant.  (Rows 32 bytes
// apart in the banks cost both reads twice the cycles, 16 bytes the transposing one four times.)
template <int D>
struct Tile {
  static constexpr int kPieces = D / 8;                       // of a row
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kCopies = kTrainTile * kPieces / 64;   // of a tile
  static constexpr int kSteps = D / 16;                       // of a product over the channels
  static constexpr int kBlocks = D / 32;                      // channel blocks of a result
  // where copy c starts, the row that lane `lane` of it holds, and where a row is; `at` is a sum over the bits of the row
  static constexpr __device__ __forceinline__ int copy_at(int c) { return D == 128 ? c * 1088 + c / 4 * 16 : c * 1088 + c / 2 * 144; }
  static constexpr __device__ __forceinline__ int row_of(int c, int lane) {
    const int slot = lane / kPieces;
    return D == 128 ? c + 16 * slot : (c & 1) + 2 * (slot & 1) + 4 * (c >> 1) + 16 * (slot >> 1);
  }
  static constexpr __device__ __forceinline__ int at(int r) {
    return D == 128 ? copy_at(r & 15) + (r >> 4) * kRowBytes : copy_at((r & 1) + 2 * (r >> 2 & 3)) + ((r >> 1 & 1) + 2 * (r >> 4)) * kRowBytes;
  }
  static constexpr int kBytes = (copy_at(kCopies - 1) + 1024 + 63) / 64 * 64;
};

// lds_copy16 (sage_attn_device.h) with the destination as the LDS address it is
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_copy16_at(const void* base, unsigned lane_off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(lane_off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lds_copy4_at(const void* base, unsigned lane_off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(lane_off), "s"(base) : "memory", "m0");
}
// .. from an address of each lane's own
__device__ __forceinline__ void lds_copy16_from(const void* lane_at, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(lane_at) : "memory", "m0");
}
#pragma clang diagnostic pop
// All copies of this wave but the youngest kLater are in LDS, its LDS reads are done, and so are the other waves'.
template <int kLater>
__device__ __forceinline__ void tile_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLater) : "memory");
}

typedef const __attribute__((address_space(3))) v4i* LdsV4;
typedef const __attribute__((address_space(3))) v4f* LdsF4;
typedef __attribute__((address_space(3))) v4s* LdsS4;

// The eight values of row 32 block + m, channels 16 step + 8 hh ..: `lane_at` of the lane, and constants
template <int D>
__device__ __forceinline__ unsigned row_lane_at(int lane) {
  return Tile<D>::at(lane & 31) + (lane >> 5) * 16;
}
template <int D>
__device__ __forceinline__ v4i read_row(unsigned tile_and_lane, int block, int step) {
  return *(LdsV4)(uintptr_t)(tile_and_lane + Tile<D>::at(32 * block) + 32 * step);
}

// A's operand where the sum goes over the tile's rows: channels 32 block + m, rows 16 t + 8 (j / 4) + 4 hh + j % 4
template <int D>
__device__ __forceinline__ unsigned column_lane_at(int lane) {
  const int i = lane & 15;
  return Tile<D>::at(4 * (lane >> 5) + (i >> 2)) + (lane >> 4 & 1) * 32 + (i & 3) * 8;
}
template <int D>
__device__ __forceinline__ v4i read_column(unsigned tile_and_lane, int block, int t) {
  const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(uintptr_t)(tile_and_lane + Tile<D>::at(16 * t) + 64 * block)));
  const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(uintptr_t)(tile_and_lane + Tile<D>::at(16 * t + 8) + 64 * block)));
  return v4i{lo[0], lo[1], hi[0], hi[1]};
}

// Query rows of the heads that share a key head, numbered together: row r is position r / group of head r % group.
__device__ __forceinline__ int row_position(const TrainAttnParams& p, int r) {
  return p.group == 1 ? r : (int)__umulhi((unsigned)r, p.group_inv);
}
__device__ __forceinline__ int64_t row_offset(const TrainAttnParams& p, const TrainTensor& t, int r) {
  const int l = row_position(p, r);
  return (int64_t)l * t.sL + (int64_t)(r - l * p.group) * t.sH;
}

// A wave's copies of tiles of a tensor's rows.  Of a whole tile they are one lane offset and addresses that the wave shares; of one with
// fewer rows, those that do not exist are copies of the last one: they are finite where the tensor is, and what the products make of
// them is not looked at.
template <int D, int kWaves>
struct TileCopy {
  using T = Tile<D>;
  const char* base;      // of the head
  int64_t row_bytes;
  unsigned whole;        // the lane's offset in a whole tile
  __device__ __forceinline__ TileCopy(const uint16_t* head, int64_t sL, int wave, int lane)
      : base(reinterpret_cast<const char*>(head)), row_bytes(sL * 2),
        whole((unsigned)T::row_of(wave, lane) * (unsigned)(sL * 2) + lane % T::kPieces * 16) {}
  // keys or values from `row` on, of which `rows` exist
  __device__ __forceinline__ void start(int row, int rows, unsigned tile, int wave, int lane) const {
    const char* at = base + row * row_bytes;
    if (rows - row >= kTrainTile) {
#pragma unroll
      for (int c = 0; c < T::kCopies / kWaves; ++c)
        lds_copy16_at(at + (T::row_of(c * kWaves, 0)) * row_bytes, whole, tile + T::copy_at(c * kWaves + wave));
    } else {
#pragma unroll
      for (int c = 0; c < T::kCopies / kWaves; ++c)
        lds_copy16_at(at, (unsigned)min(T::row_of(c * kWaves + wave, lane), rows - row - 1) * (unsigned)row_bytes + lane % T::kPieces * 16,
                      tile + T::copy_at(c * kWaves + wave));
    }
  }
  // A tile of single rows: kCount spread evenly over rows `from` to `to`, number i is from + i (to - from) / kCount, or as many as there are; then the first kCount rows.
  // Those that do not exist are copies of others.
  template <int kCount>
  __device__ __forceinline__ void start_spread(int from, int to, unsigned tile, int wave, int lane) const {
#pragma unroll
    for (int c = 0; c < T::kCopies / kWaves; ++c) {
      const int i = T::row_of(c * kWaves + wave, lane);
      const int row = i >= kCount ? i - kCount : from + (to - from >= kCount ? i * (to - from) / kCount : i);
      lds_copy16_from(base + min(row, to - 1) * row_bytes + lane % T::kPieces * 16, tile + T::copy_at(c * kWaves + wave));
    }
  }
};

// The same of query rows, numbered over the heads of a key head.  Where their number is a power of two up to 16, position and head of
// row A + B are those of A and B added (a wave's copy has one part of a row's number, a lane the other, and they share no bit), so whole
// tiles are again one lane offset and shared addresses; 16 heads of 8192 causal tokens on 4 key heads, dk and dv: 618 us, by the general way 641.
template <int D, int kWaves>
struct QueryCopy {
  using T = Tile<D>;
  const char* base;
  int64_t row_bytes, head_bytes;
  int shift;        // log2 of the number, or -1
  unsigned whole;
  __device__ __forceinline__ QueryCopy(const TrainAttnParams& p, const uint16_t* heads, const TrainTensor& t, int lane)
      : base(reinterpret_cast<const char*>(heads)), row_bytes(t.sL * 2), head_bytes(t.sH * 2), shift(p.group_shift) {
    const int of_lane = T::row_of(0, lane), by = max(shift, 0);
    whole = (unsigned)(of_lane >> by) * (unsigned)row_bytes + (unsigned)(of_lane & ((1 << by) - 1)) * (unsigned)head_bytes + lane % T::kPieces * 16;
  }
  __device__ __forceinline__ void start(const TrainAttnParams& p, int row, int rows, unsigned tile, int wave, int lane) const {
    if (shift >= 0 && rows - row >= kTrainTile) {
      const char* at = base + (row >> shift) * row_bytes;
#pragma unroll
      for (int c = 0; c < T::kCopies / kWaves; ++c) {
        const int of_copy = T::row_of(c * kWaves + wave, 0);
        lds_copy16_at(at + (of_copy >> shift) * row_bytes + (of_copy & ((1 << shift) - 1)) * head_bytes, whole, tile + T::copy_at(c * kWaves + wave));
      }
      return;
    }
    const int first = row_position(p, row);
    const char* at = base + first * row_bytes;
#pragma unroll
    for (int c = 0; c < T::kCopies / kWaves; ++c) {
      const int i = c * kWaves + wave, r = min(row + T::row_of(i, lane), rows - 1), l = row_position(p, r);
      lds_copy16_at(at, (unsigned)(l - first) * (unsigned)row_bytes + (unsigned)(r - l * p.group) * (unsigned)head_bytes + lane % T::kPieces * 16,
                    tile + T::copy_at(i));
    }
  }
};

// The largest of three, not a number if one is not (one instruction each; fmaxf on results of matrix instructions costs one more
// to make signalling values quiet)
__device__ __forceinline__ float largest(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }

// What workgroup `blockIdx.x` of a launch works on: a key head, a block of its rows or keys, and a run of the block's loop.
// Consecutive workgroups land on consecutive XCDs.  Where all blocks cost the same, every XCD takes a stretch of heads after heads, so
// that workgroups of one head share an L2.  Causal blocks and the entries of a padded batch differ: there the same block of all heads
// comes before the next block, so that XCDs share long and short ones (and still keep heads to themselves where their number is a
// multiple of eight).
struct TrainPlace {
  int bh, block, run, cut;  // cut: number of the block among those that are cut; -1: a whole block
};
__device__ __forceinline__ bool blocks_differ(const TrainAttnParams& p) { return p.causal || p.q_lens != nullptr || p.k_lens != nullptr; }
__device__ __forceinline__ TrainPlace block_place(const TrainAttnParams& p, int blocks, int i) {
  if (blocks_differ(p)) {
    const int heads = p.B * p.Hkv, block = i / heads;
    return TrainPlace{i - block * heads, block, 0, -1};
  }
  const int bh = i / blocks;
  return TrainPlace{bh, i - bh * blocks, 0, -1};
}
__device__ __forceinline__ TrainPlace train_place(const TrainAttnParams& p, int blocks) {
  const int at = (int)blockIdx.x;
  if (at < p.whole) return block_place(p, blocks, (at & 7) * (p.whole >> 3) + (at >> 3));  // (only multiples of eight are left whole)
  const int run = (at - p.whole) / p.cut, cut = at - p.whole - run * p.cut;
  TrainPlace place = block_place(p, blocks, p.whole + cut);
  place.run = run;
  place.cut = cut;
  return place;
}
// The tiles of a block's run of its tiles `first` to `last`, and how many runs it has
struct TileRange {
  int from, to, runs;
};
__device__ __forceinline__ TileRange run_tiles(const TrainAttnParams& p, const TrainPlace& place, int first, int last) {
  if (place.cut < 0) return TileRange{first, last, 1};
  const int runs = max(1, (max(0, last - first) + p.run_tiles - 1) / p.run_tiles), from = first + place.run * p.run_tiles;
  return TileRange{min(from, last), min(from + p.run_tiles, last), runs};
}

// A lane's column of a result whose rows are channels (32 dt + 8 g + 4 hh + c): two lanes hold a column's halves and exchange
// them, so that each stores runs of eight channels.
template <int DT, int D>
__device__ __forceinline__ void store_column(const v16f (&acc)[Tile<D>::kBlocks], float factor, uint16_t* row, int hh, bool store) {
#pragma unroll
  for (int b = 0; b < Tile<D>::kBlocks; ++b) {
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      const uint2 a = half4<DT>(acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor, acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor);
      const uint2 c = half4<DT>(acc[b][4 * g + 4] * factor, acc[b][4 * g + 5] * factor, acc[b][4 * g + 6] * factor, acc[b][4 * g + 7] * factor);
      const auto x = __builtin_amdgcn_permlane32_swap(a.x, c.x, false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(a.y, c.y, false, false);
      if (store) *reinterpret_cast<uint4*>(row + 32 * b + 8 * g + 8 * hh) = make_uint4(x[0], y[0], x[1], y[1]);
    }
  }
}

// .. and unrounded, for a run of a block
template <int D>
__device__ __forceinline__ void store_column_part(const v16f (&acc)[Tile<D>::kBlocks], float factor, float* row, int hh, bool store) {
  if (!store) return;
#pragma unroll
  for (int b = 0; b < Tile<D>::kBlocks; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(row + 32 * b + 8 * g + 4 * hh) =
          make_float4(acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor, acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor);
}

}  // namespace ksana_sage
