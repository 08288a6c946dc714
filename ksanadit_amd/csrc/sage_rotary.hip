// Rotary positions, and the step that fills a paged cache, which gives keys theirs on the way.
//
//   a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),  t = position frequency
//
// for the pairs (a, b) of a row's first R channels: channels 2 i and 2 i + 1, or i and i + R / 2.  The others are copied.  Backward: t negated.
//
// The angle is formed in turns in 64 bits - fp32 would be off by 2^-24 of it, 0.06 radians at a position of 10^6 - and what is left of it after its
// quarter turns are taken off goes on in 32: off by a few 2^-24, and by about 2^-52 of the angle, 2^-24 from 2^28 radians on.
//
// Bound by the rows' bytes: a workgroup forms its tokens' cosines and sines once, into LDS, and takes the rows of all heads through, the first ones asked for before.
// 32760 tokens, 2 x 40 heads of 128 channels, bf16: 227 to 235 us a direction from memory, 5.8 TB/s; of 64 channels 130, 5.2 TB/s; prompts of 16384 and 9011 tokens into
// pages, 32 + 8 + 8 heads: 130 us, 5.3 TB/s.  Few tokens are a chain of latencies: 5 us.
#include "sage_cache.h"
#include "sage_device.h"
#include "sage_train.h"

#include <algorithm>

namespace ksana_sage {

namespace {

// 16 bytes at an access, or (either order of pairs) one value, where these do not divide the head, the turned channels or, of halves, each half of them.  (32760 tokens, 2 x 16 heads
// of 80 channels of bf16, 40 of them turned: interleaved 72 us, 4.7 TB/s; halves of 20 value by value 186, 1.8 TB/s.)
enum Layout { kInterleaved, kHalves, kSingle };
template <int DT, Layout kLayout>
constexpr int kAtOnce = kLayout == kSingle ? 1 : DT == kFp32 ? 4 : 8;

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

// E values as they lie in memory (16-byte accesses at any address)
template <int DT, int E>
struct Raw {
  uint4 w;
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (E == 1)
      w.x = DT == kFp32 ? *reinterpret_cast<const uint32_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
    else
      __builtin_memcpy(&w, p, 16);
  }
  __device__ __forceinline__ void values(float (&x)[E]) const {
    if constexpr (E == 1) {
      if constexpr (DT == kFp32) x[0] = __uint_as_float(w.x);
      if constexpr (DT == KSANA_SAGE_BF16) x[0] = __uint_as_float(w.x << 16);
      if constexpr (DT == KSANA_SAGE_FP16) x[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)w.x);
    } else if constexpr (DT == kFp32) {
      __builtin_memcpy(x, &w, 16);
    } else {
      widen8<DT>(w, x);
    }
  }
};
// e4m3 as it is nearest, what lies beyond its largest number at that; not-a-numbers stay such
__device__ __forceinline__ float within_e4m3(float x) {
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}
// A head's scale, m 2^exponent with 1 / 2 <= m < 1, whatever its size
struct Scale {
  float m, inv;
  int exponent;
  __device__ __forceinline__ explicit Scale(float scale) : m(__builtin_amdgcn_frexp_mantf(scale)), inv(1.0f / m), exponent(__builtin_amdgcn_frexp_expf(scale)) {}
};
// x / scale, for a rounding to e4m3: codes, and what lies between two of them, have 19 last bits of 0 in fp32.  The product with the inverse is off by 2 in its last place at
// most, so where it is as near as that to such a number it may lie on the wrong side: the remainder, whose sign is exact, says on which.  (One value after the other: eight at
// once want more registers than there are.)  An 8-bit frame of 1560 tokens: 24.5 us, by the product alone 22.
template <int E>
__device__ __forceinline__ void divide_for_e4m3(float (&x)[E], const Scale& s) {
  constexpr uint32_t kLast = 0x7ffff;
  uint32_t least = ~0u;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = __builtin_amdgcn_ldexpf(x[e], -s.exponent);
    least = min(least, (__float_as_uint(x[e] * s.inv) + 2) & kLast);
    asm volatile("" : "+v"(x[e]), "+v"(least));
  }
  const bool some = least <= 4 && s.m != 0.5f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float y = x[e] * s.inv;
    if (some) {
      const uint32_t above = __float_as_uint(y) + 2, border = above & ~kLast;
      const float left = __fmaf_rn(-__uint_as_float(border), s.m, x[e]);
      const int side = left < 0.0f || left > 0.0f ? ((int)(__float_as_uint(left) ^ border) >> 31) | 1 : 0;  // away from 0, or to it
      y = (above & kLast) <= 4 ? __uint_as_float(border + side) : y;
    }
    x[e] = y;
    asm volatile("" : "+v"(x[e]));
  }
}
template <int DT, int E, bool kEight>
__device__ __forceinline__ void store_values(void* at, const float (&x)[E], float scale, int stream) {
  if constexpr (kEight) {
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = x[e];
    divide_for_e4m3(y, Scale(scale));
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = within_e4m3(y[e]);
    if constexpr (E == 1) {
      *static_cast<uint8_t*>(at) = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[0], 0, false);
    } else {
      uint2 w;
      w.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
      w.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false), true);
      *static_cast<uint2*>(at) = w;
    }
  } else if constexpr (E == 1) {
    if constexpr (DT == kFp32) *static_cast<float*>(at) = x[0];
    if constexpr (DT == KSANA_SAGE_BF16) *static_cast<__bf16*>(at) = (__bf16)x[0];
    if constexpr (DT == KSANA_SAGE_FP16) *static_cast<_Float16*>(at) = (_Float16)x[0];
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kFp32) {
        w[i] = __float_as_uint(x[i]);
      } else if constexpr (DT == KSANA_SAGE_BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        w[i] = __builtin_bit_cast(uint32_t, (b2){(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        w[i] = __builtin_bit_cast(uint32_t, (h2){(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
      }
    }
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    u4* to = static_cast<u4*>(at);
    if (DT != kFp32 && stream) {
      asm volatile("" ::: "memory");  // (the two are made one otherwise, before or behind the branch, and that is not the first)
      __builtin_nontemporal_store(u4{w[0], w[1], w[2], w[3]}, to);
      asm volatile("" ::: "memory");
    } else {
      *to = u4{w[0], w[1], w[2], w[3]};
    }
  }
}

// What a workgroup holds of its tokens
struct Token {
  int there;        // in the batch's counts
  int page, slot;   // of the cache; page -1: not stored
};
constexpr int kMostTokens = 16;

// A workgroup takes a few tokens: first its threads form a cosine and a sine each, of a pair of a token, then all rows go through, a thread with E channels at `lo`
// and E at `hi` of every one, neighbours beside each other.  (Every thread forming what it needs itself, eight pairs for three rows: 360 us
// of 32760 tokens, 2 x 40 heads, where this takes 230.)  Seven waves to a SIMD: with six the 1560 workgroups of a frame in 8 bits take a round more, 27.4 us for 24.6, and with eight
// registers go through memory, 27.5.
template <int DT, Layout kLayout, bool kCache, bool kEight>
__global__ __launch_bounds__(256, 7) void sage_rotary_kernel(const RotaryParams p) {
  constexpr int E = kAtOnce<DT, kLayout>, kAhead = 2;
  extern __shared__ __align__(16) float2 turns[];  // [tokens][R / 2]: cosine and sine
  __shared__ Token token_of[kMostTokens];
  const int pairs = p.R / 2, all = p.B * p.L, token0 = (int)blockIdx.x * p.tokens_each, tokens = min(p.tokens_each, all - token0), rows = tokens * p.heads;
  const int unit = (int)threadIdx.x % p.units, slot = (int)threadIdx.x / p.units;
  // where the unit lies, and the numbers of its pairs
  int lo, hi, pair_lo, pair_hi;
  bool turn_lo, turn_hi;
  if constexpr (kLayout == kInterleaved) {
    lo = E * unit;
    hi = E * (unit + p.units);
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
      lo = p.R + E * rest;
      hi = lo + E * (p.units - turned);
    }
  }
  const bool has_hi = hi < p.D;
  const int apart = kLayout == kInterleaved ? E * p.units : hi - lo;

  struct Row {
    int t, part, head;
    bool is;
    Raw<DT, E> x, y;
  } row[kAhead];
  // A field of a row's part, by value: a reference that differs from lane to lane is read from memory, field by field, into registers that the rows need.
  auto of = [&](int part, auto q, auto k, auto v) { return kCache && part == 2 ? v : part == 1 ? k : q; };
  // (Rows behind the counts are read as others where L is 1, whatever is made of them: their entry's count would be waited for first.)
  const bool counted = kCache && p.pages.q_lens != nullptr && p.L > 1;
  auto fetch = [&](int first) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      Row& r = row[n];
      const int number = first + n * p.slots;
      r.is = number < rows;
      r.t = quotient(min(number, rows - 1), p.by_heads);
      r.head = min(number, rows - 1) - r.t * p.heads;
      r.part = r.head < p.part[0].H ? 0 : r.head < p.part[0].H + p.part[1].H ? 1 : 2;
      r.head -= r.part == 0 ? 0 : r.part == 1 ? p.part[0].H : p.part[0].H + p.part[1].H;
      const int b = quotient(token0 + r.t, p.by_length), l = token0 + r.t - b * p.L;
      const RotaryPart *q = p.part, *k = p.part + 1, *v = p.part + 2;
      const char* at = static_cast<const char*>(of(r.part, q->src, k->src, v->src)) +
                       (b * of(r.part, q->sB, k->sB, v->sB) + l * of(r.part, q->sL, k->sL, v->sL) + r.head * of(r.part, q->sH, k->sH, v->sH) + lo) * kWidth<DT>;
      r.x = r.y = Raw<DT, E>{};
      if (r.is && (!counted || l < p.pages.q_lens[b])) {
        r.x.load(at);
        if (has_hi) r.y.load(at + apart * kWidth<DT>);
      }
    }
  };
  const bool works = slot < p.slots;
  if (works) fetch(slot);

  auto place_of = [&](int b, int l, int& n) {
    n = p.L;
    if constexpr (kCache) {
      if (p.pages.q_lens != nullptr) n = rows_counted(p.pages.q_lens[b], p.L);
      return (int)((int64_t)max(p.pages.k_lens[b], 0) - n + l);
    }
    return l;
  };
  for (int i = (int)threadIdx.x; i < tokens * pairs; i += 256) {
    const int t = i / pairs, pair = i - t * pairs, b = quotient(token0 + t, p.by_length), l = token0 + t - b * p.L;
    double position;
    if (p.positions != nullptr) {
      int axis = 0;
#pragma unroll
      for (int a = 1; a < kMostAxes; ++a) axis = a < p.axes && pair >= p.ends[a - 1] ? a : axis;
      const int64_t offset = b * p.pos_sB + l * p.pos_sL + axis * p.pos_sA;
      position = p.pos64 ? (double)static_cast<const int64_t*>(p.positions)[offset] : (double)static_cast<const int32_t*>(p.positions)[offset];
    } else {
      int n;
      position = (double)place_of(b, l, n);
    }
    float c, s;
    turn_of(position, p.frequencies[pair], c, s);
    turns[i] = make_float2(c * p.magnitude, s * (p.inverse ? -p.magnitude : p.magnitude));
  }
  if (kCache && (int)threadIdx.x < tokens) {
    const int t = (int)threadIdx.x, b = quotient(token0 + t, p.by_length), l = token0 + t - b * p.L;
    int n;
    const int place = place_of(b, l, n);
    Token own{l < n, -1, 0};
    if (own.there && place >= 0) {
      const int number = quotient(place, p.pages.size);
      own.slot = place - number * p.pages.size.by;
      if (number < p.pages.width) {
        const int page = p.pages.table[b * p.pages.sB + number];
        own.page = (unsigned)page < (unsigned)p.pages.pages ? page : -1;
      }
    }
    token_of[t] = own;
  }
  __syncthreads();
  if (!works) return;

  for (int first = slot; first < rows; first += kAhead * p.slots) {
    if (first != slot) fetch(first);
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const Row& r = row[n];
      if (!r.is) continue;
      const bool paged = kCache && r.part > 0;
      Token token{1, 0, 0};
      if constexpr (kCache) token = token_of[r.t];
      if (paged && token.page < 0) continue;
      float x[E], y[E];
      r.x.values(x);
      r.y.values(y);
      if (kCache && !token.there) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = y[e] = 0.0f;
      }
      if (!kCache || r.part < 2) {
        const float2* own = turns + r.t * pairs;
        if constexpr (kLayout == kInterleaved) {
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            if (turn_lo) {
              const float2 z = own[pair_lo + e];
              const float a = x[2 * e];
              x[2 * e] = __fmaf_rn(a, z.x, -x[2 * e + 1] * z.y);
              x[2 * e + 1] = __fmaf_rn(a, z.y, x[2 * e + 1] * z.x);
            }
            if (turn_hi) {
              const float2 z = own[pair_hi + e];
              const float a = y[2 * e];
              y[2 * e] = __fmaf_rn(a, z.x, -y[2 * e + 1] * z.y);
              y[2 * e + 1] = __fmaf_rn(a, z.y, y[2 * e + 1] * z.x);
            }
          }
        } else if (turn_lo) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float2 z = own[pair_lo + e];
            const float a = x[e];
            x[e] = __fmaf_rn(a, z.x, -y[e] * z.y);
            y[e] = __fmaf_rn(a, z.y, y[e] * z.x);
          }
        }
      }
      if (paged) {
        constexpr int kSize = kEight ? 1 : kWidth<DT>;
        const RotaryPart &k = p.part[1], &v = p.part[2];  // (laid out alike)
        char* at = static_cast<char*>(r.part == 1 ? k.dst : v.dst) + (token.page * k.dB + token.slot * k.dL + r.head * k.dH + lo) * kSize;
        const float* scales = r.part == 1 ? k.scale : v.scale;
        const float scale = kEight && scales != nullptr ? scales[r.head] : 1.0f;
        store_values<DT, E, kEight>(at, x, scale, p.stream);
        if (has_hi) store_values<DT, E, kEight>(at + apart * kSize, y, scale, p.stream);
      } else {
        const RotaryPart &q = p.part[0], &k = p.part[1];
        const bool second = !kCache && r.part == 1;
        char* at = static_cast<char*>(second ? k.dst : q.dst) + (((int64_t)(token0 + r.t) * (second ? k.H : q.H) + r.head) * p.D + lo) * kWidth<DT>;
        store_values<DT, E, false>(at, x, 1.0f, p.stream);
        if (has_hi) store_values<DT, E, false>(at + apart * kWidth<DT>, y, 1.0f, p.stream);
      }
    }
  }
}

template <int DT, Layout kLayout>
void start(const RotaryParams& p, unsigned groups, hipStream_t s) {
  const unsigned lds = (unsigned)(p.tokens_each * (p.R / 2) * 8);
  if (p.pages.table == nullptr) {
    sage_rotary_kernel<DT, kLayout, false, false><<<groups, 256, lds, s>>>(p);
  } else if constexpr (DT != kFp32) {
    if (p.eight_bits)
      sage_rotary_kernel<DT, kLayout, true, true><<<groups, 256, lds, s>>>(p);
    else
      sage_rotary_kernel<DT, kLayout, true, false><<<groups, 256, lds, s>>>(p);
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
  const int at_once = p.dtype == kFp32 ? 4 : 8;
  if (p.D % at_once == 0 && p.R % (p.interleaved ? at_once : 2 * at_once) == 0) layout = p.interleaved ? kInterleaved : kHalves;
  p.heads = p.part[0].H + p.part[1].H + p.part[2].H;
  p.units = layout == kInterleaved ? (p.D / at_once + 1) / 2
            : layout == kHalves    ? p.R / (2 * at_once) + (p.D - p.R + 2 * at_once - 1) / (2 * at_once)
                                   : p.R / 2 + (p.D - p.R + 1) / 2;
  // 16-bit results go first out of the caches, as what has been read, where an access of neighbours fills whole lines.  32760 tokens, 2 x 40 heads of 128: 236 us, kept
  // like others 247; of 64 channels 139 and 130; of 80, 32 of them turned, 222 and 155.
  const int piece = layout == kInterleaved ? p.units * 16 : p.R;
  p.stream = layout != kSingle && p.dtype != kFp32 && piece % 128 == 0 && (layout == kInterleaved ? p.D == 16 * p.units : p.R == p.D);
  p.slots = 256 / p.units;  // rows at a time
  p.by_heads = divisor(p.heads);
  p.by_length = divisor(p.L);
  // About three rows to a thread where that leaves four workgroups to each of 256 compute units.  32760 tokens, 2 x 40 heads: of one token 234 us, of
  // two 254, of four 266, of sixteen 278; two prompts, 48 heads: 143, 132, 133, 157; a frame in 8 bits of one 24.5, of more 29.6.
  const int tokens = p.B * p.L;
  p.tokens_each = std::max({1, std::min({kMostTokens, 3 * p.slots / p.heads, (tokens + 1023) / 1024}), (tokens + (1 << 23) - 1) >> 23});  // (a launch has fewer than 2^32 threads)
  const unsigned groups = (unsigned)((tokens + p.tokens_each - 1) / p.tokens_each);
  if (p.dtype == KSANA_SAGE_BF16)
    start_layout<KSANA_SAGE_BF16>(p, layout, groups, s);
  else if (p.dtype == KSANA_SAGE_FP16)
    start_layout<KSANA_SAGE_FP16>(p, layout, groups, s);
  else
    start_layout<kFp32>(p, layout, groups, s);
  return hipGetLastError();
}

}  // namespace ksana_sage
