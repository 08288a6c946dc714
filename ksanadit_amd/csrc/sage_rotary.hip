// Rotary positions, and the step that fills a paged cache, which gives keys theirs on the way.
//
//   a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),  t = position frequency
//
// for the pairs (a, b) of a row's first R channels: channels 2 i and 2 i + 1, or i and i + R / 2.  The others are copied.  Backward: t negated.
//
// The angle is formed in turns in 64 bits - fp32 would be off by 2^-24 of it, 0.06 radians at a position of 10^6 - and what is left of it after its
// quarter turns are taken off goes on in 32.  Bound by the rows' bytes: a thread keeps the cosines and sines of sixteen channels of a token and takes its
// heads' rows through one after the other.
#include "sage_cache.h"
#include "sage_device.h"
#include "sage_train.h"

#include <algorithm>

namespace ksana_sage {

namespace {

enum Layout { kInterleaved, kHalves, kSingle };  // eight channels at an access, or (either order of pairs) one

// cos and sin of x / 4 turns for |x| <= 1 / 2, by their series: the first terms left out are below 2e-9 and 2e-10 there
__device__ __forceinline__ void quarter_turn(float x, float& c, float& s) {
  const float t = x * 1.57079632679489662f, u = t * t;
  s = __fmaf_rn(__fmaf_rn(__fmaf_rn(__fmaf_rn(1.0f / 362880.0f, u, -1.0f / 5040.0f), u, 1.0f / 120.0f), u, -1.0f / 6.0f) * u, t, t);
  c = __fmaf_rn(__fmaf_rn(__fmaf_rn(__fmaf_rn(__fmaf_rn(-1.0f / 3628800.0f, u, 1.0f / 40320.0f), u, -1.0f / 720.0f), u, 1.0f / 24.0f), u, -0.5f), u, 1.0f);
}
__device__ __forceinline__ void turn_of(double position, double frequency, float& c, float& s) {
  double t = position * frequency * 0.15915494309189533577;
  t = 4.0 * (t - rint(t));
  const double whole = rint(t);
  float a, b;
  quarter_turn((float)(t - whole), a, b);
  const int q = (int)whole & 3;
  c = q == 0 ? a : q == 1 ? -b : q == 2 ? -a : b;
  s = q == 0 ? b : q == 1 ? a : q == 2 ? -b : -a;
}

template <int DT>
constexpr int kWidth = DT == kFp32 ? 4 : 2;

template <int DT, int E>
__device__ __forceinline__ void load_values(const void* row, int64_t at, float (&x)[E]) {
  if constexpr (E == 1) {
    if constexpr (DT == kFp32) x[0] = static_cast<const float*>(row)[at];
    if constexpr (DT == KSANA_SAGE_BF16) x[0] = __uint_as_float((uint32_t)static_cast<const uint16_t*>(row)[at] << 16);
    if constexpr (DT == KSANA_SAGE_FP16) x[0] = (float)static_cast<const _Float16*>(row)[at];
  } else {  // (16-byte accesses at any address)
    const char* p = static_cast<const char*>(row) + at * kWidth<DT>;
    if constexpr (DT == kFp32) {
      __builtin_memcpy(x, p, 16);
      __builtin_memcpy(x + 4, p + 16, 16);
    } else {
      uint4 raw;
      __builtin_memcpy(&raw, p, 16);
      widen8<DT>(raw, x);
    }
  }
}
// e4m3 as it is nearest, what lies beyond its largest number at that; not-a-numbers stay such
__device__ __forceinline__ float within_e4m3(float x) {
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}
template <int DT, int E, bool kEight>
__device__ __forceinline__ void store_values(void* row, int64_t at, const float (&x)[E], float inv) {
  if constexpr (kEight) {
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = within_e4m3(x[e] * inv);
    if constexpr (E == 1) {
      static_cast<uint8_t*>(row)[at] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[0], 0, false);
    } else {
      uint2 w;
      w.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
      w.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false), true);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(row) + at) = w;
    }
  } else if constexpr (E == 1) {
    if constexpr (DT == kFp32) static_cast<float*>(row)[at] = x[0];
    if constexpr (DT == KSANA_SAGE_BF16) static_cast<__bf16*>(row)[at] = (__bf16)x[0];
    if constexpr (DT == KSANA_SAGE_FP16) static_cast<_Float16*>(row)[at] = (_Float16)x[0];
  } else if constexpr (DT == kFp32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == KSANA_SAGE_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        w[i] = __builtin_bit_cast(uint32_t, (b2){(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        w[i] = __builtin_bit_cast(uint32_t, (h2){(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A thread's unit: E channels at `lo` and E at `hi` of a row; units up to `turned` are turned whole or by group (interleaved).
template <int DT, Layout kLayout, bool kCache, bool kEight>
__global__ __launch_bounds__(256) void sage_rotary_kernel(const RotaryParams p) {
  constexpr int E = kLayout == kSingle ? 1 : 8;
  const int unit = (int)threadIdx.x % p.units, slot = (int)threadIdx.x / p.units;
  if (slot >= p.head_slots * p.token_slots) return;
  const int head0 = slot % p.head_slots, token0 = slot / p.head_slots;
  // where the unit lies, and the numbers of its pairs
  int lo, hi, pair_lo, pair_hi;
  bool turn_lo, turn_hi;
  if constexpr (kLayout == kInterleaved) {
    lo = 8 * unit;
    hi = 8 * (unit + p.units);
    turn_lo = lo < p.R;
    turn_hi = hi < p.R;
    pair_lo = lo / 2;
    pair_hi = hi / 2;
  } else {
    const int turned = p.R / (2 * E), rest = unit - turned;
    turn_lo = turn_hi = rest < 0;
    pair_lo = E * unit;
    pair_hi = pair_lo + E / 2;
    if (kLayout == kSingle && p.interleaved) {
      lo = 2 * unit;
      hi = lo + 1;
    } else if (turn_lo) {
      lo = E * unit;
      hi = lo + p.R / 2;
    } else {
      lo = p.R + 2 * E * rest;
      hi = lo + E;
    }
  }
  const bool has_hi = hi < p.D;
  const int tokens = p.B * p.L;
  int token = (int)blockIdx.x * p.token_slots * p.tokens_each + token0;
  for (int i = 0; i < p.tokens_each && token < tokens; ++i, token += p.token_slots) {
    const int b = token / p.L, l = token - b * p.L;
    int place = l;
    bool there = true, stored = false;
    int page = 0, in_page = 0;
    if constexpr (kCache) {
      const int n = p.pages.q_lens != nullptr ? rows_counted(p.pages.q_lens[b], p.L) : p.L;
      place = (int)((int64_t)max(p.pages.k_lens[b], 0) - n + l);
      there = l < n;
      if (there && place >= 0) {
        const int number = quotient(place, p.pages.size);
        in_page = place - number * p.pages.size.by;
        if (number < p.pages.width) {
          page = p.pages.table[b * p.pages.sB + number];
          stored = (unsigned)page < (unsigned)p.pages.pages;
        }
      }
    }
    float c[E], s[E];
    if (turn_lo || turn_hi) {
      double at[kMostAxes];
#pragma unroll
      for (int a = 0; a < kMostAxes; ++a) {
        at[a] = (double)place;
        if (p.positions != nullptr && a < p.axes) {
          const int64_t offset = b * p.pos_sB + l * p.pos_sL + a * p.pos_sA;
          at[a] = p.pos64 ? (double)static_cast<const int64_t*>(p.positions)[offset] : (double)static_cast<const int32_t*>(p.positions)[offset];
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        // (a group that is not turned has no pairs: the last one's then, and nothing is made of them)
        const int pair = min(e < (E + 1) / 2 ? pair_lo + e : pair_hi + e - (E + 1) / 2, p.R / 2 - 1);
        double position = at[0];
#pragma unroll
        for (int a = 1; a < kMostAxes; ++a) position = a < p.axes && pair >= p.ends[a - 1] ? at[a] : position;
        turn_of(position, p.frequencies[pair], c[e], s[e]);
        c[e] *= p.magnitude;
        s[e] *= p.inverse ? -p.magnitude : p.magnitude;
      }
    }
    for (int h = head0; h < p.heads; h += p.head_slots) {
      int head = h;
      const bool second = head >= p.part[0].H;
      head -= second ? p.part[0].H : 0;
      const bool third = second && head >= p.part[1].H;
      head -= third ? p.part[1].H : 0;
      const RotaryPart& part = third ? p.part[2] : second ? p.part[1] : p.part[0];
      float x[E], y[E];
      if (kCache && !there) {
        if (part.paged) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = y[e] = 0.0f;
      } else {
        if (kCache && part.paged && !stored) continue;
        const char* row = static_cast<const char*>(part.src) + (b * part.sB + l * part.sL + head * part.sH) * kWidth<DT>;
        load_values<DT, E>(row, lo, x);
        if (has_hi) load_values<DT, E>(row, hi, y);
        if (part.turn) {
          if constexpr (kLayout == kInterleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = x[2 * e], d = y[2 * e];
              if (turn_lo) {
                x[2 * e] = __fmaf_rn(a, c[e], -x[2 * e + 1] * s[e]);
                x[2 * e + 1] = __fmaf_rn(a, s[e], x[2 * e + 1] * c[e]);
              }
              if (turn_hi) {
                y[2 * e] = __fmaf_rn(d, c[4 + e], -y[2 * e + 1] * s[4 + e]);
                y[2 * e + 1] = __fmaf_rn(d, s[4 + e], y[2 * e + 1] * c[4 + e]);
              }
            }
          } else if (turn_lo) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float a = x[e];
              x[e] = __fmaf_rn(a, c[e], -y[e] * s[e]);
              y[e] = __fmaf_rn(a, s[e], y[e] * c[e]);
            }
          }
        }
      }
      if (kCache && part.paged) {
        constexpr int kSize = kEight ? 1 : kWidth<DT>;
        char* row = static_cast<char*>(part.dst) + (page * part.dB + in_page * part.dL + head * part.dH) * kSize;
        const float inv = kEight && part.scale != nullptr ? 1.0f / part.scale[head] : 1.0f;
        store_values<DT, E, kEight>(row, lo, x, inv);
        if (has_hi) store_values<DT, E, kEight>(row, hi, y, inv);
      } else {
        char* row = static_cast<char*>(part.dst) + (b * part.dB + l * part.dL + head * part.dH) * kWidth<DT>;
        store_values<DT, E, false>(row, lo, x, 1.0f);
        if (has_hi) store_values<DT, E, false>(row, hi, y, 1.0f);
      }
    }
  }
}

template <int DT, Layout kLayout>
void start(const RotaryParams& p, unsigned groups, hipStream_t s) {
  if (p.pages.table == nullptr) {
    sage_rotary_kernel<DT, kLayout, false, false><<<groups, 256, 0, s>>>(p);
  } else if constexpr (DT != kFp32) {
    if (p.eight_bits)
      sage_rotary_kernel<DT, kLayout, true, true><<<groups, 256, 0, s>>>(p);
    else
      sage_rotary_kernel<DT, kLayout, true, false><<<groups, 256, 0, s>>>(p);
  }
}
template <int DT>
void start_layout(const RotaryParams& p, Layout layout, unsigned groups, hipStream_t s) {
  if (layout == kInterleaved)
    start<DT, kInterleaved>(p, groups, s);
  else if (layout == kHalves)
    start<DT, kHalves>(p, groups, s);
  else
    start<DT, kSingle>(p, groups, s);
}

}  // namespace

hipError_t launch_rotary(RotaryParams p, hipStream_t s) {
  Layout layout = kSingle;
  if (p.D % 8 == 0 && p.R % (p.interleaved ? 8 : 16) == 0) layout = p.interleaved ? kInterleaved : kHalves;
  p.heads = p.part[0].H + p.part[1].H + p.part[2].H;
  p.units = layout == kInterleaved ? (p.D / 8 + 1) / 2 : layout == kHalves ? p.R / 16 + (p.D - p.R + 15) / 16 : p.R / 2 + (p.D - p.R + 1) / 2;
  // rows at a time: those of a token's heads, spread evenly over its passes, and of as many tokens as there is place for
  const int slots = 256 / p.units, passes = (p.heads + slots - 1) / slots;
  p.head_slots = (p.heads + passes - 1) / passes;
  p.token_slots = slots / p.head_slots;
  p.tokens_each = 1;
  const int64_t tokens = (int64_t)p.B * p.L;
  const unsigned groups = (unsigned)((tokens + (int64_t)p.token_slots * p.tokens_each - 1) / ((int64_t)p.token_slots * p.tokens_each));
  if (p.dtype == KSANA_SAGE_BF16)
    start_layout<KSANA_SAGE_BF16>(p, layout, groups, s);
  else if (p.dtype == KSANA_SAGE_FP16)
    start_layout<KSANA_SAGE_FP16>(p, layout, groups, s);
  else
    start_layout<kFp32>(p, layout, groups, s);
  return hipGetLastError();
}

}  // namespace ksana_sage
