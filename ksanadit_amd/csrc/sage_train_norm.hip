// What stands between two parts of a block, in one pass over the residual stream x and the part's output y, with its backward pass:
//
//   u = post(y) post_weight                   (u = y without a norm behind the part)
//   h = residual_scale x + gate u
//   n = (norm(h) weight + bias) (1 + scale) + shift
//
// norm and post: layer (mean and variance) or rms over the C channels of a row.  gate, scale and shift are vectors of C channels for
// every batch entry or for all.  With a = weight (1 + scale), G = gate post_weight, hat the normalised row, N' the norm's derivative:
//
//   dh' = dh + N'(dn a)      dx = residual_scale dh'      d(post(y)) = dh' G
//   S0 = sum dn,  S1 = sum dn hat,  K = sum dh' post(y)  over the rows of a batch entry, from which all vectors' gradients follow:
//   d shift = S0,  d scale = weight S1 + bias S0,  d gate = post_weight K,
//   d weight = sum_b (1 + scale) S1,  d bias = sum_b (1 + scale) S0,  d post_weight = sum_b gate K
//
// Everything is bound by the bytes of x, y and the results: a workgroup keeps its columns' vectors (and, backward, their three sums)
// in registers and walks rows of one batch entry, the next row's loads in flight.  The sums of the workgroups are added in a fixed
// order by a second launch.  All arithmetic is fp32; each result is rounded once.
#include "sage_device.h"
#include "sage_train.h"

#include <algorithm>

namespace ksana_sage {

namespace {

template <int DT>
struct Raw {  // eight values as they lie in memory
  uint4 w[DT == kFp32 ? 2 : 1];
};
template <int DT>
constexpr int kSize = DT == kFp32 ? 4 : 2;

template <int DT>
__device__ __forceinline__ void store_one(void* p, int64_t i, float x) {
  if constexpr (DT == kFp32) static_cast<float*>(p)[i] = x;
  if constexpr (DT == KSANA_SAGE_BF16) static_cast<__bf16*>(p)[i] = (__bf16)x;
  if constexpr (DT == KSANA_SAGE_FP16) static_cast<_Float16*>(p)[i] = (_Float16)x;
}
__device__ __forceinline__ float load_any(const TrainVector& v, int b, int c) {
  const int64_t i = b * v.sB + c;
  if (v.dtype == kFp32) return static_cast<const float*>(v.ptr)[i];
  if (v.dtype == KSANA_SAGE_BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t*>(v.ptr)[i] << 16);
  return (float)static_cast<const _Float16*>(v.ptr)[i];
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float x) {
  if (dtype == kFp32)
    store_one<kFp32>(p, i, x);
  else if (dtype == KSANA_SAGE_BF16)
    store_one<KSANA_SAGE_BF16>(p, i, x);
  else
    store_one<KSANA_SAGE_FP16>(p, i, x);
}

// A thread's columns of a row: 8 (v T + thread) .., T the workgroup's threads, eight at an access whatever the row's address (the GPU takes
// 16-byte accesses at any).  kWhole: C is a multiple of eight.  Else a row's last eight columns overlap those before: both threads compute and
// store the same values there, and sums leave out the second one's (`own`).  Value by value instead, 8331 rows of 1153 took 57 us
// forward and 157 backward where this takes 25 and 45.
template <bool kWhole, int kVecs>
struct Columns {
  int C, T, thread;
  __device__ __forceinline__ int due(int v) const { return 8 * (v * T + thread); }
  __device__ __forceinline__ bool some(int v) const { return due(v) < C; }
  __device__ __forceinline__ int first(int v) const { return kWhole ? due(v) : max(0, min(due(v), C - 8)); }
  __device__ __forceinline__ bool own(int v, int e) const { return kWhole ? some(v) : some(v) && first(v) + e >= due(v) && first(v) + e < C; }

  template <int DT>
  __device__ __forceinline__ void load(const void* row, Raw<DT> (&raw)[kVecs]) const {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      raw[v] = Raw<DT>{};
      if (!some(v)) continue;
      const char* p = static_cast<const char*>(row) + (int64_t)first(v) * kSize<DT>;
      if (kWhole || C >= 8) {
        __builtin_memcpy(&raw[v].w[0], p, 16);
        if constexpr (DT == kFp32) __builtin_memcpy(&raw[v].w[1], p + 16, 16);
      } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(&raw[v]);
        for (int e = 0; e < C; ++e) {
          uint32_t x;
          if constexpr (DT == kFp32)
            x = reinterpret_cast<const uint32_t*>(p)[e];
          else
            x = (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
#pragma unroll
          for (int i = 0; i < (DT == kFp32 ? 8 : 4); ++i) w[i] |= i == (DT == kFp32 ? e : e >> 1) ? x : 0u;
        }
      }
    }
  }
  template <int DT>
  static __device__ __forceinline__ void widen(const Raw<DT>& raw, float (&x)[8]) {
    if constexpr (DT == kFp32) {
      const uint32_t w[8] = {raw.w[0].x, raw.w[0].y, raw.w[0].z, raw.w[0].w, raw.w[1].x, raw.w[1].y, raw.w[1].z, raw.w[1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
    } else {
      widen8<DT>(raw.w[0], x);
    }
  }
  template <int DT, bool kStream = true>
  __device__ __forceinline__ void store(void* row, int v, const float (&x)[8]) const {
    if (!some(v)) return;
    char* p = static_cast<char*>(row) + (int64_t)first(v) * kSize<DT>;
    if (kWhole || C >= 8) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8 / (4 / kSize<DT>); ++i) {
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
      // First out of the caches: the rows that come next and the next call's are worth more of them.  8704 rows of 5120 fp32 channels 102 us,
      // kept like others 113; 32760 bf16 rows backward 402 and 416; with a reader of both results right behind, 1560 rows 34.0 and
      // 34.9, 8192 rows 119 and 113, 16384 rows 230 and 237.
      typedef int Piece __attribute__((ext_vector_type(4), aligned(2)));
      const Piece lo = {(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
      if constexpr (kStream)
        __builtin_nontemporal_store(lo, reinterpret_cast<Piece*>(p));
      else
        *reinterpret_cast<Piece*>(p) = lo;
      if constexpr (DT == kFp32) {
        const Piece hi = {(int)w[4], (int)w[5], (int)w[6], (int)w[7]};
        if constexpr (kStream)
          __builtin_nontemporal_store(hi, reinterpret_cast<Piece*>(p + 16));
        else
          *reinterpret_cast<Piece*>(p + 16) = hi;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < C) store_one<DT>(p, e, x[e]);
    }
  }
  // A vector's values, `otherwise` where there is none
  struct Vector {
    Raw<kFp32> raw[kVecs];
    __device__ __forceinline__ void load(const Columns& c, const TrainVector& vec, int b) {
      if (vec.ptr == nullptr) return;
      const char* at = static_cast<const char*>(vec.ptr) + b * vec.sB * (vec.dtype == kFp32 ? 4 : 2);
      if (vec.dtype == kFp32) {
        c.load<kFp32>(at, raw);
      } else {
        Raw<KSANA_SAGE_BF16> half[kVecs];
        c.load<KSANA_SAGE_BF16>(at, half);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) raw[v].w[0] = half[v].w[0];
      }
    }
    __device__ __forceinline__ void values(const TrainVector& vec, float otherwise, int v, float (&x)[8]) const {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = otherwise;
      if (vec.ptr == nullptr) return;
      if (vec.dtype == kFp32) {
        widen<kFp32>(raw[v], x);
      } else if (vec.dtype == KSANA_SAGE_BF16) {
        widen8<KSANA_SAGE_BF16>(raw[v].w[0], x);
      } else {
        widen8<KSANA_SAGE_FP16>(raw[v].w[0], x);
      }
    }
  };
};

constexpr int kMaxThreads = 512, kMaxWaves = kMaxThreads / 64;

// Two sums over a workgroup.  `turn` alternates between two places in LDS, so that one barrier per call is enough: a wave that is back
// here for the place's next use has passed the barrier between, and with it every wave has read the place.
struct Sums {
  float a, b;
};
__device__ __forceinline__ Sums workgroup_sums(Sums x, int waves, int& turn, float (*lds)[kMaxWaves][2]) {
  x.a = over_lanes<Sum>(x.a);
  x.b = over_lanes<Sum>(x.b);
  if (waves == 1) return x;
  if ((threadIdx.x & 63) == 0) {
    lds[turn][threadIdx.x >> 6][0] = x.a;
    lds[turn][threadIdx.x >> 6][1] = x.b;
  }
  __syncthreads();
  Sums all{0.0f, 0.0f};
  for (int w = 0; w < waves; ++w) {
    all.a += lds[turn][w][0];
    all.b += lds[turn][w][1];
  }
  turn ^= 1;
  return all;
}

struct RowStats {
  float mean, inv;
};
// Mean (layer) and 1 / sqrt(variance or mean square + eps) of a row.  The variance is the sum of the squares about each wave's own mean
// and of what the waves' means differ by: no cancellation, and one barrier.
template <bool kWhole, int kVecs>
__device__ __forceinline__ RowStats row_stats(const Columns<kWhole, kVecs>& c, const float (&x)[kVecs][8], int kind, float eps, int waves, int& turn,
                                              float (*lds)[kMaxWaves][2]) {
  const float n = (float)c.C;
  if (kind == kNormRms) {
    float square = 0.0f;
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) square = c.own(v, e) ? __fmaf_rn(x[v][e], x[v][e], square) : square;
    const float all = workgroup_sums(Sums{square, 0.0f}, waves, turn, lds).a;
    return RowStats{0.0f, 1.0f / sqrtf(all / n + eps)};
  }
  float sum = 0.0f;
  int own = 0;
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum += c.own(v, e) ? x[v][e] : 0.0f;
      own += c.own(v, e) ? 1 : 0;
    }
  sum = over_lanes<Sum>(sum);
  const float count = over_lanes<Sum>((float)own);
  const float wave_mean = count > 0.0f ? sum / count : 0.0f;
  float square = 0.0f;
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = c.own(v, e) ? x[v][e] - wave_mean : 0.0f;
      square = __fmaf_rn(d, d, square);
    }
  square = over_lanes<Sum>(square);
  if (waves == 1) return RowStats{wave_mean, 1.0f / sqrtf(square / n + eps)};
  // (the counts of the waves' columns follow from their numbers: only the sums are exchanged)
  __shared__ float counts[kMaxWaves];
  if ((threadIdx.x & 63) == 0) {
    lds[turn][threadIdx.x >> 6][0] = wave_mean;
    lds[turn][threadIdx.x >> 6][1] = square;
    counts[threadIdx.x >> 6] = count;  // (the same in every row)
  }
  __syncthreads();
  float mean = 0.0f, all = 0.0f;
  for (int w = 0; w < waves; ++w) mean = __fmaf_rn(lds[turn][w][0], counts[w], mean);
  mean /= n;
  for (int w = 0; w < waves; ++w) {
    const float d = lds[turn][w][0] - mean;
    all += __fmaf_rn(d * d, counts[w], lds[turn][w][1]);
  }
  turn ^= 1;
  return RowStats{mean, 1.0f / sqrtf(all / n + eps)};
}

// A workgroup's rows: a stretch of one batch entry's
struct RowRange {
  int b, from, to;
};
__device__ __forceinline__ RowRange row_range(const TrainNormParams& p) {
  const int b = (int)blockIdx.x / p.groups, g = (int)blockIdx.x - b * p.groups;
  const int from = min(p.L, g * p.rows_each);
  return RowRange{b, from, min(p.L, from + p.rows_each)};
}

template <int XT, int YT, bool kWhole, int kVecs>
__global__ __launch_bounds__(kMaxThreads) void sage_train_norm_fwd_kernel(const TrainNormParams p) {
  __shared__ float lds[2][kMaxWaves][2];
  const Columns<kWhole, kVecs> c{p.C, (int)blockDim.x, (int)threadIdx.x};
  const int waves = (int)blockDim.x >> 6;
  int turn = 0;
  const RowRange rows = row_range(p);
  if (rows.from >= rows.to) return;
  const char* x_at = static_cast<const char*>(p.x) + (rows.b * p.x_sB + rows.from * p.x_sL) * kSize<XT>;
  const char* y_at = static_cast<const char*>(p.y) + (rows.b * p.y_sB + rows.from * p.y_sL) * kSize<YT>;
  const bool has_y = p.y != nullptr;
  // Two rows on their way while one is worked on: 32760 rows of 5120 bf16 channels 276 us, 4.9 TB/s, with one row on its way 383.  (A copy
  // reaches 5.0.)  fp32 rows beside bf16 ones, 8704 of 5120: 97 us, 5.5 TB/s: more than a copy's, part of what
  // is read is in the last-level cache still when a call follows another on the same rows.
  struct Rows {
    Raw<XT> x[kVecs];
    Raw<YT> y[kVecs];
  } raw[2] = {};
  int fetched = rows.from;
  auto fetch = [&](Rows& into) {
    if (fetched >= rows.to) return;
    c.template load<XT>(x_at, into.x);
    if (has_y) c.template load<YT>(y_at, into.y);
    x_at += p.x_sL * kSize<XT>;
    y_at += p.y_sL * kSize<YT>;
    ++fetched;
  };
  fetch(raw[0]);
  fetch(raw[1]);
  float a[kVecs][8], t[kVecs][8], g[kVecs][8];
  {
    typename Columns<kWhole, kVecs>::Vector weight, bias, scale, shift, gate, post_weight;  // (all on their way before the first is used)
    weight.load(c, p.weight, rows.b);
    scale.load(c, p.scale, rows.b);
    bias.load(c, p.bias, rows.b);
    shift.load(c, p.shift, rows.b);
    gate.load(c, p.gate, rows.b);
    post_weight.load(c, p.post_weight, rows.b);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      float w[8], bs[8], sc[8], sh[8], ga[8], po[8];
      weight.values(p.weight, 1.0f, v, w);
      scale.values(p.scale, 0.0f, v, sc);
      bias.values(p.bias, 0.0f, v, bs);
      shift.values(p.shift, 0.0f, v, sh);
      gate.values(p.gate, 1.0f, v, ga);
      post_weight.values(p.post_weight, 1.0f, v, po);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[v][e] = w[e] * (1.0f + sc[e]);
        t[v][e] = bs[e] * (1.0f + sc[e]) + sh[e];
        g[v][e] = has_y ? ga[e] * po[e] : 0.0f;
      }
    }
  }
  const int64_t first = (int64_t)rows.b * p.L;
  auto work = [&](int row, Rows& from) {
    float h[kVecs][8], y[kVecs][8];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      c.template widen<XT>(from.x[v], h[v]);
      c.template widen<YT>(from.y[v], y[v]);
    }
    fetch(from);
    // (no norm behind the part: mean 0 and factor 1, no y: a gate of 0)
    RowStats of_y{0.0f, 1.0f};
    if (p.post != kNormNone) of_y = row_stats(c, y, p.post, p.eps, waves, turn, lds);
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = __fmaf_rn(g[v][e], (y[v][e] - of_y.mean) * of_y.inv, p.residual_scale * h[v][e]);
    const RowStats of_h = row_stats(c, h, p.norm, p.eps, waves, turn, lds);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (p.h != nullptr) c.template store<XT>(static_cast<char*>(p.h) + (first + row) * p.C * kSize<XT>, v, h[v]);
      float n[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = __fmaf_rn((h[v][e] - of_h.mean) * of_h.inv, a[v][e], t[v][e]);
      c.template store<YT>(static_cast<char*>(p.n) + (first + row) * p.C * kSize<YT>, v, n);
    }
    if (p.stats != nullptr && threadIdx.x == 0)
      *reinterpret_cast<float4*>(p.stats + 4 * (first + row)) = make_float4(of_h.mean, of_h.inv, of_y.mean, of_y.inv);
  };
  for (int row = rows.from; row < rows.to; row += 2) {
    work(row, raw[0]);
    if (row + 1 < rows.to) work(row + 1, raw[1]);
  }
}

// Reads x, y, dh and dn again rather than keep normalised rows: 32760 rows of 5120 bf16 channels 400 us, 5.0 TB/s.
template <int XT, int YT, bool kWhole, int kVecs>
__global__ __launch_bounds__(kMaxThreads) void sage_train_norm_bwd_kernel(const TrainNormParams p) {
  __shared__ float lds[2][kMaxWaves][2];
  const Columns<kWhole, kVecs> c{p.C, (int)blockDim.x, (int)threadIdx.x};
  const int waves = (int)blockDim.x >> 6;
  int turn = 0;
  const RowRange rows = row_range(p);
  const bool has_y = p.y != nullptr, has_dh = p.dh != nullptr;
  const int64_t first = (int64_t)rows.b * p.L;
  float s0[kVecs][8], s1[kVecs][8], kk[kVecs][8];
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) s0[v][e] = s1[v][e] = kk[v][e] = 0.0f;
  if (rows.from < rows.to) {
    const char* x_at = static_cast<const char*>(p.x) + (rows.b * p.x_sB + rows.from * p.x_sL) * kSize<XT>;
    const char* y_at = static_cast<const char*>(p.y) + (rows.b * p.y_sB + rows.from * p.y_sL) * kSize<YT>;
    const char* dh_at = static_cast<const char*>(p.dh) + (first + rows.from) * p.C * kSize<XT>;
    const char* dn_at = static_cast<const char*>(p.dn) + (first + rows.from) * p.C * kSize<YT>;
    Raw<XT> x_raw[kVecs], dh_raw[kVecs] = {};
    Raw<YT> y_raw[kVecs] = {}, dn_raw[kVecs];
    c.template load<XT>(x_at, x_raw);
    if (has_y) c.template load<YT>(y_at, y_raw);
    if (has_dh) c.template load<XT>(dh_at, dh_raw);
    c.template load<YT>(dn_at, dn_raw);
    float4 stats = *reinterpret_cast<const float4*>(p.stats + 4 * (first + rows.from));
    float a[kVecs][8], g[kVecs][8];
    {
      typename Columns<kWhole, kVecs>::Vector weight, scale, gate, post_weight;
      weight.load(c, p.weight, rows.b);
      scale.load(c, p.scale, rows.b);
      gate.load(c, p.gate, rows.b);
      post_weight.load(c, p.post_weight, rows.b);
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        float w[8], sc[8], ga[8], po[8];
        weight.values(p.weight, 1.0f, v, w);
        scale.values(p.scale, 0.0f, v, sc);
        gate.values(p.gate, 1.0f, v, ga);
        post_weight.values(p.post_weight, 1.0f, v, po);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[v][e] = w[e] * (1.0f + sc[e]);
          g[v][e] = has_y ? ga[e] * po[e] : 0.0f;
        }
      }
    }
    const float n = (float)p.C;
    for (int row = rows.from; row < rows.to; ++row) {
      const RowStats of_h{stats.x, stats.y}, of_y{stats.z, stats.w};
      float hat[kVecs][8], y[kVecs][8], d[kVecs][8], m[kVecs][8];  // the normalised row, u (without its weight), dh, dn
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        c.template widen<XT>(x_raw[v], hat[v]);
        c.template widen<YT>(dn_raw[v], m[v]);
        c.template widen<XT>(dh_raw[v], d[v]);
        c.template widen<YT>(y_raw[v], y[v]);
      }
      if (row + 1 < rows.to) {
        x_at += p.x_sL * kSize<XT>;
        y_at += p.y_sL * kSize<YT>;
        dh_at += (int64_t)p.C * kSize<XT>;
        dn_at += (int64_t)p.C * kSize<YT>;
        c.template load<XT>(x_at, x_raw);
        if (has_y) c.template load<YT>(y_at, y_raw);
        if (has_dh) c.template load<XT>(dh_at, dh_raw);
        c.template load<YT>(dn_at, dn_raw);
        stats = *reinterpret_cast<const float4*>(p.stats + 4 * (first + row + 1));
      }
      Sums sums{0.0f, 0.0f};  // of dn a hat and of dn a
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[v][e] = (y[v][e] - of_y.mean) * of_y.inv;
          hat[v][e] = (__fmaf_rn(g[v][e], y[v][e], p.residual_scale * hat[v][e]) - of_h.mean) * of_h.inv;
          s0[v][e] += m[v][e];
          s1[v][e] = __fmaf_rn(m[v][e], hat[v][e], s1[v][e]);
          m[v][e] *= a[v][e];
          sums.a = c.own(v, e) ? __fmaf_rn(m[v][e], hat[v][e], sums.a) : sums.a;
          sums.b += c.own(v, e) ? m[v][e] : 0.0f;
        }
      sums = workgroup_sums(sums, waves, turn, lds);
      const float along = sums.a / n, mean = p.norm == kNormLayer ? sums.b / n : 0.0f;
      Sums of_post{0.0f, 0.0f};
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          d[v][e] = __fmaf_rn(of_h.inv, m[v][e] - mean - hat[v][e] * along, d[v][e]);
          kk[v][e] = __fmaf_rn(d[v][e], y[v][e], kk[v][e]);
          const float through = d[v][e] * g[v][e];
          hat[v][e] = d[v][e] * p.residual_scale;
          d[v][e] = through;
          if (c.own(v, e)) {
            of_post.a = __fmaf_rn(through, y[v][e], of_post.a);
            of_post.b += through;
          }
        }
        c.template store<XT>(static_cast<char*>(p.dx) + (first + row) * p.C * kSize<XT>, v, hat[v]);
      }
      if (p.dy == nullptr) continue;
      float y_along = 0.0f, y_mean = 0.0f;
      if (p.post != kNormNone) {
        of_post = workgroup_sums(of_post, waves, turn, lds);
        y_along = of_post.a / n;
        y_mean = p.post == kNormLayer ? of_post.b / n : 0.0f;
      }
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] = of_y.inv * (d[v][e] - y_mean - y[v][e] * y_along);
        c.template store<YT>(static_cast<char*>(p.dy) + (first + row) * p.C * kSize<YT>, v, d[v]);
      }
    }
  }
  float* part = p.part + (int64_t)blockIdx.x * 3 * p.C;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    c.template store<kFp32, false>(part, v, s0[v]);
    c.template store<kFp32, false>(part + p.C, v, s1[v]);
    c.template store<kFp32, false>(part + 2 * p.C, v, kk[v]);
  }
}

// The workgroups' sums added up, 16 columns to a workgroup, its 64 groups of threads sharing the parts; and what follows from the sums.
// Bound by latency: everything a thread reads of an entry (24 values of up to 512 parts) is on its way before the first is added.  One entry of
// 5120 columns 10 us, three of 1153 12 us.
constexpr int kJoinColumns = 16, kSlots = 64, kAtOnce = 8;
__global__ __launch_bounds__(1024) void sage_train_norm_vectors_kernel(const TrainNormParams p) {
  constexpr int kWaves = kJoinColumns * kSlots / 64;
  __shared__ float lds[2][3][kWaves][kJoinColumns];
  const int lane = threadIdx.x % kJoinColumns, slot = threadIdx.x / kJoinColumns, column = min((int)blockIdx.x * kJoinColumns + lane, p.C - 1);
  const bool writes = slot == 0 && (int)blockIdx.x * kJoinColumns + lane < p.C;
  float d_gate = 0.0f, d_scale = 0.0f, d_shift = 0.0f, d_weight = 0.0f, d_bias = 0.0f, d_post = 0.0f;
  for (int b = 0; b < p.B; ++b) {
    float w = 1.0f, bias = 0.0f, s = 1.0f, gate = 1.0f, post = 1.0f;
    if (slot == 0) {
      if (p.weight.ptr != nullptr) w = load_any(p.weight, b, column);
      if (p.bias.ptr != nullptr) bias = load_any(p.bias, b, column);
      if (p.scale.ptr != nullptr) s = 1.0f + load_any(p.scale, b, column);
      if (p.gate.ptr != nullptr) gate = load_any(p.gate, b, column);
      if (p.post_weight.ptr != nullptr) post = load_any(p.post_weight, b, column);
    }
    const float* part = p.part + (int64_t)b * p.groups * 3 * p.C + column;
    float sum[3] = {};
    for (int first = slot; first < p.groups; first += kSlots * kAtOnce) {
      float x[kAtOnce][3];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
        for (int i = 0; i < 3; ++i) x[j][i] = part[((int64_t)min(first + j * kSlots, p.groups - 1) * 3 + i) * p.C];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
        for (int i = 0; i < 3; ++i) sum[i] += first + j * kSlots < p.groups ? x[j][i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      sum[i] += __shfl_xor(sum[i], 16);
      sum[i] += __shfl_xor(sum[i], 32);
      if ((threadIdx.x & 63) < kJoinColumns) lds[b & 1][i][threadIdx.x >> 6][lane] = sum[i];
    }
    __syncthreads();  // (the two places alternate: one barrier an entry)
    if (slot != 0) continue;
    float all[3] = {};
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int v = 0; v < kWaves; ++v) all[i] += lds[b & 1][i][v][lane];
    const float of_gate = post * all[2], of_scale = __fmaf_rn(w, all[1], bias * all[0]);
    const int64_t at = (int64_t)b * p.C + column;
    if (writes) {  // vectors of every entry's own
      if (p.d_gate != nullptr && p.gate.sB != 0) store_any(p.d_gate, p.gate.dtype, at, of_gate);
      if (p.d_scale != nullptr && p.scale.sB != 0) store_any(p.d_scale, p.scale.dtype, at, of_scale);
      if (p.d_shift != nullptr && p.shift.sB != 0) store_any(p.d_shift, p.shift.dtype, at, all[0]);
    }
    d_gate += of_gate;
    d_scale += of_scale;
    d_shift += all[0];
    d_weight = __fmaf_rn(s, all[1], d_weight);
    d_bias = __fmaf_rn(s, all[0], d_bias);
    d_post = __fmaf_rn(gate, all[2], d_post);
  }
  if (!writes) return;
  if (p.d_gate != nullptr && p.gate.sB == 0) store_any(p.d_gate, p.gate.dtype, column, d_gate);
  if (p.d_scale != nullptr && p.scale.sB == 0) store_any(p.d_scale, p.scale.dtype, column, d_scale);
  if (p.d_shift != nullptr && p.shift.sB == 0) store_any(p.d_shift, p.shift.dtype, column, d_shift);
  if (p.d_weight != nullptr) store_any(p.d_weight, p.weight.dtype, column, d_weight);
  if (p.d_bias != nullptr) store_any(p.d_bias, p.bias.dtype, column, d_bias);
  if (p.d_post_weight != nullptr) store_any(p.d_post_weight, p.post_weight.dtype, column, d_post);
}

// ------------------------------------------------------------------------------------------------------------ launches

struct NormShape {
  int vecs, threads;
};
NormShape norm_shape(int C) {
  for (int vecs = 1; vecs <= 2; ++vecs) {  // (with three, the backward kernel's sums and rows do not fit the registers; with two, 2 - 10 of fp32 streams of odd width go through memory)
    const int threads = (C + 512 * vecs - 1) / (512 * vecs) * 64;
    if (threads <= kMaxThreads) return NormShape{vecs, threads};
  }
  return NormShape{0, 0};
}

// Workgroups of a batch entry and their rows: about as many workgroups in all as the GPU holds at once.  Its 256 compute units hold 16
// and 12 waves each of the forward kernels with one and two pieces to a thread, 12 and 8 of the backward kernels.
void deal_rows(TrainNormParams& p, bool backward) {
  const NormShape shape = norm_shape(p.C);
  const int waves = shape.threads / 64, room = (shape.vecs == 1 ? 16 : 12) - (backward ? 4 : 0), places = 256 * std::max(1, room / waves);
  const int groups = std::max(1, std::min(p.L, places / p.B));
  p.rows_each = (p.L + groups - 1) / groups;
  p.groups = (p.L + p.rows_each - 1) / p.rows_each;
}

template <int XT, int YT, bool kWhole, int kVecs>
void start(const TrainNormParams& p, bool backward, hipStream_t s) {
  const dim3 grid((unsigned)(p.B * p.groups)), block(norm_shape(p.C).threads);
  if (backward)
    sage_train_norm_bwd_kernel<XT, YT, kWhole, kVecs><<<grid, block, 0, s>>>(p);
  else
    sage_train_norm_fwd_kernel<XT, YT, kWhole, kVecs><<<grid, block, 0, s>>>(p);
}
template <int XT, int YT>
void start(const TrainNormParams& p, bool backward, hipStream_t s) {
  switch (norm_shape(p.C).vecs + (p.C % 8 == 0 ? 0 : 4)) {
    case 1: return start<XT, YT, true, 1>(p, backward, s);
    case 2: return start<XT, YT, true, 2>(p, backward, s);
    case 5: return start<XT, YT, false, 1>(p, backward, s);
    default: return start<XT, YT, false, 2>(p, backward, s);
  }
}
hipError_t launch(const TrainNormParams& p, bool backward, hipStream_t s) {
  if (p.x_dtype == kFp32 && p.y_dtype == kFp32)
    start<kFp32, kFp32>(p, backward, s);
  else if (p.x_dtype == kFp32 && p.y_dtype == KSANA_SAGE_BF16)
    start<kFp32, KSANA_SAGE_BF16>(p, backward, s);
  else if (p.x_dtype == kFp32)
    start<kFp32, KSANA_SAGE_FP16>(p, backward, s);
  else if (p.x_dtype == KSANA_SAGE_BF16)
    start<KSANA_SAGE_BF16, KSANA_SAGE_BF16>(p, backward, s);
  else
    start<KSANA_SAGE_FP16, KSANA_SAGE_FP16>(p, backward, s);
  return hipGetLastError();
}

}  // namespace

bool train_norm_width_fits(int C) { return norm_shape(C).vecs != 0; }

uint64_t train_norm_scratch(TrainNormParams p) {
  deal_rows(p, true);
  return (uint64_t)p.B * p.groups * 3 * p.C * 4;
}

hipError_t launch_train_norm_fwd(TrainNormParams p, hipStream_t s) {
  deal_rows(p, false);
  return launch(p, false, s);
}

hipError_t launch_train_norm_bwd(TrainNormParams p, void* scratch, hipStream_t s) {
  deal_rows(p, true);
  p.part = static_cast<float*>(scratch);
  const hipError_t e = launch(p, true, s);
  if (e != hipSuccess) return e;
  sage_train_norm_vectors_kernel<<<(p.C + kJoinColumns - 1) / kJoinColumns, kJoinColumns * kSlots, 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace ksana_sage
