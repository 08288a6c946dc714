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

// A tile: 64 rows of D 16-bit channels, 16-byte pieces, a row's pieces exchanged by an exclusive or with a number of the row, so that
// neither lanes that read one piece of 32 rows nor lanes that read two pieces of four rows (the transposing read) meet in a
// bank.  The copies into LDS are linear there: a lane fetches the piece that belongs where it writes.
template <int D>
struct Tile {
  static constexpr int kPieces = D / 8;                       // of a row
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kBytes = kTrainTile * kRowBytes;
  static constexpr int kRowsPerCopy = 64 / kPieces;           // one copy instruction of a wave: 1 KiB
  static constexpr int kCopies = kBytes / 1024;               // of a tile
  static constexpr int kSteps = D / 16;                       // of a product over the channels
  static constexpr int kBlocks = D / 32;                      // channel blocks of a result
  static __device__ __forceinline__ int twist(int row) {
    return D == 128 ? ((row & 7) << 1 | (row >> 3 & 1)) : ((row >> 1 & 3) << 1 | (row >> 3 & 1));
  }
};

// lds_copy16 (sage_attn_device.h) with the destination as the LDS address it is
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_copy16_at(const void* base, unsigned lane_off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(lane_off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void lds_copy4_at(const void* base, unsigned lane_off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(lds), "v"(lane_off), "s"(base) : "memory", "m0");
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

// The eight values of rows 32 block + m: byte offsets in a tile of the lane's piece of step s = at[s] + block * 32 rows
template <int D>
struct RowReader {
  unsigned at[Tile<D>::kSteps];
  __device__ __forceinline__ explicit RowReader(int lane) {
    const int row = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int s = 0; s < Tile<D>::kSteps; ++s) at[s] = row * Tile<D>::kRowBytes + (((2 * s + hh) ^ Tile<D>::twist(row)) << 4);
  }
  __device__ __forceinline__ v4i read(unsigned tile, int block, int s) const {
    return *(LdsV4)(uintptr_t)(tile + at[s] + block * 32 * Tile<D>::kRowBytes);
  }
};

// A's operand where the sum goes over the tile's rows: channels 32 block + m, rows 16 t + 8 (j / 4) + 4 hh + j % 4
template <int D>
struct ColumnReader {
  unsigned at[2][Tile<D>::kBlocks];
  __device__ __forceinline__ explicit ColumnReader(int lane) {
    const int hh = lane >> 5, half = lane >> 4 & 1, i = lane & 15;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * j + 4 * hh + (i >> 2);
#pragma unroll
      for (int b = 0; b < Tile<D>::kBlocks; ++b) {
        const int piece = 4 * b + 2 * half + (i >> 1 & 1);
        at[j][b] = row * Tile<D>::kRowBytes + ((piece ^ Tile<D>::twist(row)) << 4) + (i & 1) * 8;
      }
    }
  }
  __device__ __forceinline__ v4i read(unsigned tile, int block, int t) const {
    const unsigned step = tile + t * 16 * Tile<D>::kRowBytes;
    const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(uintptr_t)(step + at[0][block])));
    const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(uintptr_t)(step + at[1][block])));
    return v4i{lo[0], lo[1], hi[0], hi[1]};
  }
};

// Query rows of the heads that share a key head, numbered together: row r is position r / group of head r % group.
__device__ __forceinline__ int row_position(const TrainAttnParams& p, int r) {
  return p.group == 1 ? r : (int)__umulhi((unsigned)r, p.group_inv);
}
__device__ __forceinline__ int64_t row_offset(const TrainAttnParams& p, const TrainTensor& t, int r) {
  const int l = row_position(p, r);
  return (int64_t)l * t.sL + (int64_t)(r - l * p.group) * t.sH;
}

// Starts a wave's share of the copy of 64 rows of keys or values from `row` on, of which `rows` exist.  Rows that do not are
// copies of the last one: they are finite where the tensor is, and what the products make of them is not looked at.
template <int D, int kWaves>
__device__ __forceinline__ void copy_key_tile(const uint16_t* head, int64_t sL, int row, int rows, unsigned tile, int wave, int lane) {
  using T = Tile<D>;
  const char* base = reinterpret_cast<const char*>(head + (int64_t)row * sL);
  const unsigned row_bytes = (unsigned)(sL * 2);
  const int left = rows - row - 1;
#pragma unroll
  for (int c = 0; c < T::kCopies / kWaves; ++c) {
    const int r = (c * kWaves + wave) * T::kRowsPerCopy + lane / T::kPieces;
    const int piece = (lane % T::kPieces) ^ T::twist(r);
    lds_copy16_at(base, (unsigned)min(r, left) * row_bytes + piece * 16, tile + (c * kWaves + wave) * 1024);
  }
}
// .. and of query rows, numbered as above
template <int D, int kWaves>
__device__ __forceinline__ void copy_query_tile(const TrainAttnParams& p, const uint16_t* heads, const TrainTensor& t, int row, int rows, unsigned tile,
                                                int wave, int lane) {
  using T = Tile<D>;
  const int first = row_position(p, row);
  const char* base = reinterpret_cast<const char*>(heads + (int64_t)first * t.sL);
  const unsigned l_bytes = (unsigned)(t.sL * 2), h_bytes = (unsigned)(t.sH * 2);
#pragma unroll
  for (int c = 0; c < T::kCopies / kWaves; ++c) {
    const int i = (c * kWaves + wave) * T::kRowsPerCopy + lane / T::kPieces;
    const int piece = (lane % T::kPieces) ^ T::twist(i);
    const int r = min(row + i, rows - 1), l = row_position(p, r);
    lds_copy16_at(base, (unsigned)(l - first) * l_bytes + (unsigned)(r - l * p.group) * h_bytes + piece * 16, tile + (c * kWaves + wave) * 1024);
  }
}

// Number `blockIdx.x` of a launch of a multiple of eight workgroups.  Consecutive ones land on consecutive XCDs: every XCD takes a run
// of the work, so that workgroups of one head share an L2.
__device__ __forceinline__ int xcd_run_number() { return (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3); }

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

}  // namespace ksana_sage
