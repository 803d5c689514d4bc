// From the partial statistics of the logits to losses: shared by the kernel
// that does this for many rows and the few-rows kernel's last block.
#pragma once

#include "losses.cuh"

namespace po {

// Rows of packed operands are zero up to a multiple of this (a K block of the
// 16-bit products), so that dW's last K block adds nothing.
constexpr int kRowPad = 128;

// Device-side state of a call.
struct CallState {
  int count;         // counted rows
  int counted_mean;  // rows that the mean divides by
  int done;          // blocks of the finishing launch that are through
  float alpha;       // the upstream factor that all rows share
  float alpha_dh, alpha_dw;  // the products' factors: it, with the powers of two of operand and result
  float grad_max;    // max |row_grad|
  // fp16 gradients:
  float coef_max;    // largest |1 + 2 z_loss lse| of the rows finished so far, 1 at least
  float store_dh, store_dw;  // powers of two that the gradients of a mean are stored by (0: not chosen yet)
  float redo_dh, redo_dw;    // what earlier launches' gradients are multiplied by to agree with these
  int splits;        // of K in the next dH product
};

// Cost of `s` splits of K for a product's tiles, in 16-bit K blocks (~0.6 us):
// the tiles' waves over the pairs of SMs, each tile paying its blocks and about
// 3 more to fill and drain, plus the join's traffic (8 bytes a value and split
// at ~5 TB/s).
__host__ __device__ inline float split_cost(int s, int tiles, int nkb, float values, int pairs) {
  const int waves = (tiles * s + pairs - 1) / pairs;
  const float cost = static_cast<float>(waves) * (static_cast<float>((nkb + s - 1) / s) + 3.0f);
  return s > 1 ? cost + 5.0f + static_cast<float>(s) * values * (8.0f / 3.0e6f) : cost;
}

// The split of dH's K is chosen again from the counted rows, which fill fewer
// tiles than the rows the host knows of. A pass of 50257 x 768, the host's
// choice against this one: bf16, 410 of 2048 rows 233 / 186 us, 410 of 1024 186
// / 176, fp32, 400 of 1000 757 / 680; all rows counted: the same.
struct SplitArgs {
  int nkb;     // K blocks (0: the host's choice stays)
  int tiles_n, dim, pairs;
  int units;   // tiles times splits that the workspace holds
};

struct FinishArgs {
  SplitArgs split;
  const float2* part;
  const float* zsum;
  int nparts;
  int row0, rows;
  const int* rowmap;
  const float* zpick;
  const int* ent;
  const float* q;      // nullable: hard targets
  const float* qlogq;
  int top;
  float smoothing, z_loss, temperature, inv_vocab, scale2;
  float4* stat;        // [row of this launch] max, 1 / sum, log sum exp at temperature 1
  float* loss_rows;
  float* loss;         // nullable; written by the last block of the last launch
  long long T;
  int mean, final_launch;
  CallState* st;
  uint4* packed;       // 16-byte words of H's packed rows of this launch (and of their low halves, nullable)
  uint4* packed_lo;
  int row_words;
};

// One warp: maximum and sum of a packed row from its partial statistics, and its
// loss. The statistics' maxima are the logits' own; a difference of two logits
// is scaled, never a logit. (Loads bypass L1: other SMs wrote, perhaps in this launch.)
__device__ __forceinline__ void finish_row(const FinishArgs& a, int row, int lane) {
  const float2* p = a.part + static_cast<long long>(row) * a.nparts;
  float m = -INFINITY, s = 0.0f;
  for (int i0 = lane; i0 < a.nparts; i0 += 8 * 32) {  // eight loads in flight
    float2 v[8];
    float c = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * 32;
      v[u] = i < a.nparts ? __ldcg(p + i) : make_float2(-INFINITY, 0.0f);
      c = fmaxf(c, v[u].x);
    }
    if (c > m) {
      s *= ex2((m - c) * a.scale2);
      m = c;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      s += v[u].x == -INFINITY ? v[u].y : v[u].y * ex2((v[u].x - m) * a.scale2);  // an empty part holds 0, or a NaN to keep
  }
  const float mm = warp_max(m);
  s = warp_sum(m == -INFINITY ? s : s * ex2((m - mm) * a.scale2));
  const float logs = logf(s), lse = mm + logs;
  const long long t = a.rowmap[a.row0 + row];
  float zs = 0.0f;
  if (a.zsum != nullptr) {
    for (int i = lane; i < a.nparts; i += 32) zs += __ldcg(a.zsum + static_cast<long long>(row) * a.nparts + i);
    zs = warp_sum(zs);
  }
  float loss;
  if (a.q == nullptr) {
    const float zy = __ldcg(a.zpick + t);
    loss = logs + (mm - zy) + a.z_loss * lse * lse;
    if (a.smoothing != 0.0f) loss += a.smoothing * (zy - zs * a.inv_vocab);
  } else {
    float c = 0.0f;
    for (int k = lane; k < a.top; k += 32) {
      const float q = a.q[t * a.top + k];
      if (q != 0.0f) c += q * (logs + (mm - __ldcg(a.zpick + t * a.top + k)) / a.temperature);
    }
    c = warp_sum(c);
    loss = a.temperature * a.temperature * (a.qlogq[t] + c);
  }
  if (lane == 0) {
    // (fp16 operands are scaled by it; a row without a finite one has no finite gradient)
    const float coef = fabsf(1.0f + 2.0f * a.z_loss * lse);
    if (a.z_loss != 0.0f && coef < INFINITY) atomicMax(reinterpret_cast<int*>(&a.st->coef_max), __float_as_int(coef));
    a.stat[row] = make_float4(mm, 1.0f / s, lse, 0.0f);
    a.loss_rows[t] = loss;
  }
}

// One warp: a packed row of zeros.
__device__ __forceinline__ void zero_row(const FinishArgs& a, int row, int lane) {
  if (a.packed == nullptr) return;
  const uint4 none = make_uint4(0, 0, 0, 0);
  for (int i = lane; i < a.row_words; i += 32) {
    a.packed[static_cast<long long>(row) * a.row_words + i] = none;
    if (a.packed_lo != nullptr) a.packed_lo[static_cast<long long>(row) * a.row_words + i] = none;
  }
}

// The whole block: the sum of all rows' losses in a fixed order (fp64).
__device__ __forceinline__ void finish_total(const FinishArgs& a, double* dbuf) {
  double sum = 0.0;
  for (long long t0 = threadIdx.x; t0 < a.T; t0 += 8 * blockDim.x) {  // eight loads in flight
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = t0 + u * blockDim.x < a.T ? __ldcg(a.loss_rows + t0 + u * blockDim.x) : 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += static_cast<double>(v[u]);
  }
  sum = block_sum(sum, dbuf);
  if (threadIdx.x == 0) {
    if (a.mean) sum /= static_cast<double>(a.st->counted_mean > 0 ? a.st->counted_mean : 1);
    *a.loss = static_cast<float>(sum);
  }
}

}  // namespace po
