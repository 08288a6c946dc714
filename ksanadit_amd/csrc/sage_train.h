// Launch interface of the differentiable operators (sage_train_attn.hip, sage_train_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ksana_sage {

struct TrainTensor {
  int64_t sB, sL, sH;  // element strides of [B, L, H, D]; D stride is 1
};

struct TrainAttnParams {
  const uint16_t *q, *k, *v, *d_o;
  const uint16_t* o_in;  // backward: the result
  uint16_t *o, *dq, *dk, *dv;  // dq, dk, dv: contiguous [B, L, H, D]
  float* lse;  // [B, Hq, Lq], natural logarithm; -inf where a row has no key
  TrainTensor qs, ks, vs, os, dos;
  const int32_t *q_lens, *k_lens;  // nullptr: all rows, all keys
  int dtype, B, Hq, Hkv, Lq, Lk, D, causal;
  float sm_scale;
  // filled in by the launchers
  int group;            // Hq / Hkv
  unsigned group_inv;   // ceil(2^32 / group)
  int group_shift;      // log2(group) for powers of two up to 16, else -1
  float c;              // |sm_scale| log2(e)
  uint32_t flip;        // sign bits of two 16-bit values where sm_scale is negative
  int row_pad;          // rows of row_l and row_d of a key head: Lq * group up to a multiple of 64
  float *row_l, *row_d; // backward: -log2(e) lse (-inf where a row takes no part) and -sum(dO o), [B Hkv, row_pad]
  float* norms;         // backward in fp16: largest squared norms of rows of dO and of v, [B Hkv, norm_blocks]
  int norm_blocks, norm_q_blocks;
  // of one launch: the first `whole` blocks are walked by a workgroup each, the loops of the others are cut into runs of run_tiles tiles,
  // at most `runs` of them; their results, [blocks cut, runs, 128, ..], go to `part`
  int whole, cut, runs, run_tiles;
  float* part;
};

struct TrainAttnScratch {
  uint64_t bytes, row_l, row_d, norms, part;
};

// What the launchers need of scratch memory (256-byte aligned)
TrainAttnScratch train_attn_scratch(const TrainAttnParams& p, bool backward);
hipError_t launch_train_attn_fwd(TrainAttnParams p, void* scratch, hipStream_t s);
hipError_t launch_train_attn_bwd(TrainAttnParams p, void* scratch, hipStream_t s);


// ---- residual sum, gate and norms ----

constexpr int kFp32 = 2;                                     // next to KSANA_SAGE_BF16 and _FP16
constexpr int kNormNone = 0, kNormLayer = 1, kNormRms = 2;

struct TrainVector {  // C channels, for every batch entry (sB elements apart) or for all (sB 0)
  const void* ptr;    // nullptr: none
  int64_t sB;
  int dtype;
};
struct TrainNormParams {
  int B, L, C, x_dtype, y_dtype;  // y_dtype: of y, n and their gradients
  int norm, post;
  float residual_scale, eps;
  const void *x, *y;              // y nullptr: h = x
  int64_t x_sB, x_sL, y_sB, y_sL; // in elements
  void *h, *n;                    // contiguous; h may be nullptr
  float* stats;                   // [B, L, 4]: mean and factor of h's norm and of y's
  TrainVector gate, scale, shift, weight, bias, post_weight;
  const void *dh, *dn;            // contiguous; dh may be nullptr
  void *dx, *dy;                  // contiguous; dy nullptr without y
  void *d_gate, *d_scale, *d_shift, *d_weight, *d_bias, *d_post_weight;  // of the vectors' types, contiguous [B, C] or [C], or nullptr
  // filled in by the launchers
  int groups, rows_each;          // workgroups of a batch entry, and their rows
  float* part;
};
bool train_norm_width_fits(int C);
uint64_t train_norm_scratch(TrainNormParams p);
hipError_t launch_train_norm_fwd(TrainNormParams p, hipStream_t s);
hipError_t launch_train_norm_bwd(TrainNormParams p, void* scratch, hipStream_t s);

}  // namespace ksana_sage
