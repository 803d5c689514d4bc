// Losses of a linear head over a large vocabulary, with their gradients:
// softmax cross entropy against a target, and the divergence from a teacher's
// top logits (po_linear_loss).
//
//   z = H W^T,  l_t = loss(z_t),  dZ = dl/dz,  dH = dZ W,  dW = dZ^T H
//
// Launches of one call (T rows, V vocabulary, D features):
//   targets  a teacher's rows only: q, sum q log q, indices sorted; row status
//   pack     counted rows of H packed together (a row that counts for nothing
//            costs no product, and whatever it holds reaches no sum); their
//            number stays on the device
//   logits   tensor-core product, softmax statistics in its epilogue
//            (head_gemm.cuh): 2 T V D operations
//   finish   joins each row's V / 256 statistics, writes the losses
// and with gradients
//   rescale  exp(z - max of 256 columns) -> dZ in the products' type, in place:
//            one read and one write of T V 2-byte values
//   dH, dW   two more products of 2 T V D operations
// The products bound all but the smallest calls (6 T V D operations with
// gradients). Taking the softmax apart into the tile-local exponential and a
// late factor is what makes the logits' product run once: dZ needs each row's
// sum over the whole vocabulary, which is known only after all tiles, and the
// alternative to the rescale pass (4 bytes a logit) is computing the logits
// again (2 D operations a logit).
//
// Nothing here allocates, synchronises or depends on timing: partial sums are
// joined in a fixed order.
#include <cudaTypedefs.h>

#include <climits>
#include <cmath>
#include <cstring>
#include <mutex>

#include "head_finish.cuh"
#include "head_gemm.cuh"
#include "losses.cuh"

namespace po {
namespace {

// The fp16 gradient operand is dZ / upstream times this power of two: |dZ| is at
// most 1 + |1 + 2 z_loss lse|, whose largest second term is `coef`; 2^10 keeps
// softmax values down to 6e-8 normal, and a large z-loss takes less (60000 leaves
// fp16's range a margin for the logarithm's rounding). bf16 and tf32 have fp32's
// range and need no factor.
__device__ __forceinline__ float f16_scale(float coef) {
  return fminf(1024.0f, exp2f(floorf(log2f(60000.0f / (coef + 1.0f)))));
}

struct Targets {
  const long long* index;
  long long index_ld;
  const void* teacher;
  long long teacher_ld;
  int teacher_dtype;
  int top;
  long long ignore_index;
};

// ---------------------------------------------------------------- targets
// One block a row: q = softmax(teacher / a) over the entries with index >= 0,
// sum q log q, and (index, q) sorted by index (a bitonic network over `width`
// = the next power of two; empty entries sort last as INT_MAX, q = 0). The
// maximum is subtracted before the scaling: entries of the type's lowest value
// stay finite at temperatures below 1, count, and share equally.
__global__ void teacher_targets_kernel(Targets tg, long long V, float inv_temp, int width, int* status,
                                       int* ent, float* q, float* qlogq) {
  grid_launch_next();
  grid_wait();
  extern __shared__ float sm[];
  int* si = reinterpret_cast<int*>(sm);
  float* sl = sm + width;
  __shared__ float buf[32];
  const long long t = blockIdx.x;
  float m = -INFINITY;
  bool bad = false, nan = false;
  for (int k = threadIdx.x; k < width; k += blockDim.x) {
    int i = INT_MAX;
    float l = -INFINITY;
    if (k < tg.top) {
      const long long x = tg.index[t * tg.index_ld + k];
      if (x >= V) bad = true;
      else if (x >= 0) {
        i = static_cast<int>(x);
        l = load_as_f32(tg.teacher, tg.teacher_dtype, t * tg.teacher_ld + k);
        nan |= isnan(l);
      }
    }
    si[k] = i;
    sl[k] = l;
    m = fmaxf(m, l);
  }
  bad = __syncthreads_or(bad);
  nan = __syncthreads_or(nan);
  m = block_max(m, buf);
  const int st = bad ? ROW_BAD : (m > -INFINITY || nan ? ROW_COUNTED : ROW_IGNORED);
  float sum = 0.0f;
  for (int k = threadIdx.x; k < width; k += blockDim.x)
    if (si[k] != INT_MAX) sum += expf((sl[k] - m) * inv_temp);
  sum = block_sum(sum, buf);
  const float logsum = logf(sum);
  float c = 0.0f;
  for (int k = threadIdx.x; k < width; k += blockDim.x) {
    float p = 0.0f;
    if (si[k] != INT_MAX && st == ROW_COUNTED) {
      const float d = (sl[k] - m) * inv_temp;
      p = expf(d) / sum;
      if (p != 0.0f) c += p * (d - logsum);  // NaN passes
    }
    sl[k] = p;
  }
  c = block_sum(c, buf);
  if (threadIdx.x == 0) {
    status[t] = st;
    qlogq[t] = c;
  }
  // Sort by index; the network is fixed, so equal indices land the same way each time.
  for (int size = 2; size <= width; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int k = threadIdx.x; k < width / 2; k += blockDim.x) {
        const int a = 2 * k - (k & (stride - 1)), b = a + stride;
        const bool up = (a & size) == 0;
        const int ia = si[a], ib = si[b];
        if ((ia > ib) == up && ia != ib) {
          si[a] = ib;
          si[b] = ia;
          const float f = sl[a];
          sl[a] = sl[b];
          sl[b] = f;
        }
      }
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k < tg.top; k += blockDim.x) {
    ent[t * tg.top + k] = si[k];
    q[t * tg.top + k] = sl[k];
  }
}

// ------------------------------------------------------------------- pack
struct PackArgs {
  const void* hidden;
  long long h_ld;
  long long T;
  int D, ldp;  // packed pitch (elements)
  int vec;     // 16-byte vectors on both sides
  Targets tg;
  long long V;
  const int* status;  // teacher's rows (nullable: decided by the target here)
  int* ent;           // targets (written here without a teacher)
  int* rowmap;
  void* packed;
  float* packed_lo;  // fp32: low halves of the tf32 pairs
  void* dhidden;
  long long dh_ld;
  float* loss_rows;
  CallState* st;
  unsigned int* sched;
  float alpha;
  int mean, has_row_grad;
  float* rowmax;   // nullable: max |h| of each packed row
  float* unscale;
};

__device__ __forceinline__ int row_status(const PackArgs& a, long long t, int& target) {
  if (a.status != nullptr) return a.status[t];
  const long long y = a.tg.index[t * a.tg.index_ld];
  if (y == a.tg.ignore_index) return ROW_IGNORED;
  if (y < 0 || y >= a.V) return ROW_BAD;
  target = static_cast<int>(y);
  return ROW_COUNTED;
}

// Largest finite |row_grad| of the counted rows into state->grad_max (1 when
// there is none): what stands beside the others, or one row's infinity, must not
// move the scale that all counted rows are rounded at. One block.
__global__ void grad_max_kernel(PackArgs a, const float* g) {
  grid_launch_next();
  grid_wait();
  __shared__ float buf[32];
  float m = 0.0f;
  int y;
  for (long long t = threadIdx.x; t < a.T; t += blockDim.x) {
    const float x = fabsf(g[t]);
    if (x < INFINITY && row_status(a, t, y) == ROW_COUNTED) m = fmaxf(m, x);
  }
  m = block_max(m, buf);
  if (threadIdx.x == 0) a.st->grad_max = m > 0.0f ? m : 1.0f;
}

__device__ __forceinline__ float tf32_rna(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return __uint_as_float(r);
}
// Four fp32 values as a tf32 (hi, lo) pair.
__device__ __forceinline__ void split_vec(const uint4& v, float4* hi, float4* lo) {
  const float x[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
  float h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = tf32_rna(x[i]);
    l[i] = tf32_rna(x[i] - h[i]);
  }
  *hi = make_float4(h[0], h[1], h[2], h[3]);
  *lo = make_float4(l[0], l[1], l[2], l[3]);
}


// One warp: a row of D 16-bit elements on any boundary to one on a 16-byte
// boundary, 8 elements a lane: the words around them, shifted by half a word
// where the row starts in the middle of one. Words that reach out of the row
// are not read: its first and last elements are copied one by one.
template <class T>
__device__ __forceinline__ void copy_row16(const T* src, T* dst, int D, int lane) {
  const bool odd = reinterpret_cast<uintptr_t>(src) % 4 != 0;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(src) & ~uintptr_t(3));
  const int first = odd ? 1 : 0, whole = (D - 1) / 8;  // vectors with an element of the row before and after them
#pragma unroll 4
  for (int i = first + lane; i < whole; i += 32) {
    uint32_t x[5];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = words[4 * i + k];
    x[4] = odd ? words[4 * i + 4] : 0u;
    uint4 o;
    o.x = odd ? __funnelshift_r(x[0], x[1], 16) : x[0];
    o.y = odd ? __funnelshift_r(x[1], x[2], 16) : x[1];
    o.z = odd ? __funnelshift_r(x[2], x[3], 16) : x[2];
    o.w = odd ? __funnelshift_r(x[3], x[4], 16) : x[3];
    reinterpret_cast<uint4*>(dst)[i] = o;
  }
  if (odd && lane < 8 && lane < D) dst[lane] = src[lane];
  for (int i = 8 * whole + lane; i < D; i += 32) dst[i] = src[i];
}

// Eight fp16 values.
__device__ __forceinline__ float max_abs(const uint4& v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const float2 f = __half22float2(__hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3]))));
  return fmaxf(f.x, f.y);
}

constexpr int kPackWarps = 8;

// A warp copies a row; a block takes `groups` times 8 consecutive rows. Their
// places follow from the number of counted rows before them, which the block
// counts itself (T statuses, read from L2) instead of waiting for another
// launch; the host keeps blocks x T / 2 reads small.
template <int DT>
__global__ void __launch_bounds__(32 * kPackWarps) pack_kernel(PackArgs a, int groups) {
  grid_launch_next();
  grid_wait();
  using T = typename ElemOf<DT>::T;
  __shared__ int buf[32];
  const long long first = static_cast<long long>(blockIdx.x) * groups * kPackWarps;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool last = blockIdx.x == gridDim.x - 1;
  int before = 0, bad = 0, y = 0;
  for (long long t = threadIdx.x; t < first; t += blockDim.x) {
    const int s = row_status(a, t, y);
    before += s == ROW_COUNTED;
    bad += s == ROW_BAD;
  }
  before = block_sum(before, buf);
  if (last) bad = block_sum(bad, buf);
  if (blockIdx.x == 0 && threadIdx.x < 2) a.sched[threadIdx.x] = 0u;
  T zero;
  from_f32(0.0f, zero);
  for (int g = 0; g < groups; ++g) {
    const long long t0 = first + g * kPackWarps, t = t0 + warp;
    int s = ROW_IGNORED;
    if (lane < kPackWarps && t0 + lane < a.T) s = row_status(a, t0 + lane, y);
    const unsigned votes = __ballot_sync(0xffffffffu, s == ROW_COUNTED);
    const unsigned bads = __ballot_sync(0xffffffffu, s == ROW_BAD);
    const bool counted = (votes >> warp) & 1u;
    const int place = before + __popc(votes & ((1u << warp) - 1u));
    if (lane == warp && t < a.T) {
      if (counted) a.rowmap[place] = static_cast<int>(t);
      else a.loss_rows[t] = s == ROW_BAD ? NAN : 0.0f;
      if (a.status == nullptr) a.ent[t] = counted ? y : INT_MAX;
    }
    before += __popc(votes);
    bad += __popc(bads);
    if (t >= a.T) continue;
    if (!counted) {
      if (a.dhidden != nullptr) {
        T* o = static_cast<T*>(a.dhidden) + t * a.dh_ld;
        for (int i = lane; i < a.D; i += 32) o[i] = zero;
      }
      continue;
    }
    const T* src = static_cast<const T*>(a.hidden) + t * a.h_ld;
    T* dst = static_cast<T*>(a.packed) + static_cast<long long>(place) * a.ldp;
    float* lo = DT == PO_F32 ? a.packed_lo + static_cast<long long>(place) * a.ldp : nullptr;
    constexpr int VEC = 16 / sizeof(T);
    float top = 0.0f;
    if (a.vec) {
      const int n = a.D / VEC;
      for (int i0 = lane; i0 < n; i0 += 128) {  // four loads in flight
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i0 + 32 * u < n) v[u] = reinterpret_cast<const uint4*>(src)[i0 + 32 * u];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (i0 + 32 * u >= n) continue;
          if (DT == PO_F16 && a.rowmax != nullptr) top = fmaxf(top, max_abs(v[u]));
          if (DT == PO_F32)
            split_vec(v[u], reinterpret_cast<float4*>(dst) + i0 + 32 * u, reinterpret_cast<float4*>(lo) + i0 + 32 * u);
          else reinterpret_cast<uint4*>(dst)[i0 + 32 * u] = v[u];
        }
      }
    } else if (DT == PO_F32) {
#pragma unroll 4
      for (int i = lane; i < a.D; i += 32) {
        const float v = to_f32(src[i]), h = tf32_rna(v);
        from_f32(h, dst[i]);
        lo[i] = tf32_rna(v - h);
      }
    } else {
      copy_row16(src, dst, a.D, lane);
      if (DT == PO_F16 && a.rowmax != nullptr)
        for (int i = lane; i < a.D; i += 32) top = fmaxf(top, fabsf(to_f32(src[i])));
    }
    if (DT == PO_F16 && a.rowmax != nullptr) {
      top = warp_max(top);
      if (lane == 0) a.rowmax[place] = top;
    }
  }
  if (last && threadIdx.x == 0) {
    const int all = before + bad;
    a.st->count = before;
    a.st->counted_mean = all;
    a.st->done = 0;
    float alpha = a.alpha;
    if (a.mean) alpha /= static_cast<float>(all > 0 ? all : 1);
    if (a.has_row_grad) alpha *= a.st->grad_max;
    a.st->alpha = a.st->alpha_dh = a.st->alpha_dw = alpha;
    a.st->coef_max = 1.0f;
    a.st->store_dh = a.st->store_dw = 0.0f;
    if (a.unscale != nullptr) a.unscale[0] = a.unscale[1] = 1.0f;
  }
}

// Copy of W with a pitch that TMA takes (16-bit), or as tf32 (hi, lo) pairs.
template <int DT>
__global__ void __launch_bounds__(256) stage_weight_kernel(const void* w, long long w_ld, long long V, int D, int ldp,
                                                           void* out, float* lo, int vec) {
  grid_launch_next();
  grid_wait();
  using T = typename ElemOf<DT>::T;  // (of 16-bit types only the size matters)
  if (DT == PO_F32 && vec) {
    // A thread splits 4 values; two loads in flight.
    const int n = D / 4;
    const long long total = V * n, step = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += 2 * step) {
      uint4 x[2];
      long long v[2];
      int c[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i + u * step >= total) continue;
        v[u] = (i + u * step) / n;
        c[u] = static_cast<int>(i + u * step - v[u] * n);
        x[u] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const float*>(w) + v[u] * w_ld) + c[u]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (i + u * step < total)
          split_vec(x[u], reinterpret_cast<float4*>(static_cast<float*>(out) + v[u] * ldp) + c[u],
                    reinterpret_cast<float4*>(lo + v[u] * ldp) + c[u]);
    }
    return;
  }
  if (DT != PO_F32) {  // a warp a row
    const int warps = gridDim.x * (blockDim.x >> 5);
    for (long long v = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); v < V; v += warps)
      copy_row16(static_cast<const T*>(w) + v * w_ld, static_cast<T*>(out) + v * ldp, D, threadIdx.x & 31);
    return;
  }
  for (long long v = blockIdx.x; v < V; v += gridDim.x) {
    const float* src = static_cast<const float*>(w) + v * w_ld;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      const float x = src[i], h = tf32_rna(x);
      static_cast<float*>(out)[v * ldp + i] = h;
      lo[v * ldp + i] = tf32_rna(x - h);
    }
  }
}

// ----------------------------------------------------------------- finish
// The last block to finish sums the losses of all rows. Rows past the counted
// ones are zeroed up to a K block of dW, where they meet the zeros of dZ.
constexpr int kFinishWarps = 8;

// One warp: the cheapest split for this launch's rows (the host's rule).
__device__ __forceinline__ void choose_splits(const FinishArgs& a, int left, int lane) {
  const SplitArgs& c = a.split;
  const int rows = max(1, min(a.rows, left));
  const int tiles = (rows + 255) / 256 * c.tiles_n;
  const int most = max(1, min(min(c.pairs, (c.nkb + 3) / 4), c.units / tiles));
  const float values = static_cast<float>(rows) * static_cast<float>(c.dim);
  float cost = INFINITY;
  int best = 1;
  for (int s = 1 + lane; s <= most; s += 32) {
    const float x = split_cost(s, tiles, c.nkb, values, c.pairs) * (s == 1 ? 0.98f : 1.0f);
    if (x < cost) cost = x, best = s;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, cost, o);
    const int s = __shfl_xor_sync(0xffffffffu, best, o);
    if (x < cost || (x == cost && s < best)) cost = x, best = s;
  }
  if (lane == 0) a.st->splits = best;
}

__global__ void __launch_bounds__(32 * kFinishWarps) finish_kernel(FinishArgs a) {
  grid_launch_next();
  grid_wait();
  __shared__ double dbuf[32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kFinishWarps + (threadIdx.x >> 5);
  const int left = a.st->count - a.row0;
  if (row < left && row < a.rows) finish_row(a, row, lane);
  else if (left > 0 && row < (left + kRowPad - 1) / kRowPad * kRowPad && row < (a.rows + kRowPad - 1) / kRowPad * kRowPad)
    zero_row(a, row, lane);
  if (a.split.nkb > 0 && blockIdx.x == 0 && threadIdx.x < 32) choose_splits(a, left, lane);
  if (a.loss == nullptr || !a.final_launch) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(&a.st->done, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  finish_total(a, dbuf);
}

// ---------------------------------------------------------------- rescale
struct RescaleArgs {
  void* e;        // fp16 (fp32) in, dZ of the operand type out
  float* lo;      // fp32: low halves
  long long e_ld;
  long long V;
  const float2* part;
  int nparts, part_cols;  // (64 or 256)
  const float4* stat;
  int row0, rows;
  const int* rowmap;
  const int* ent;
  const float* q;
  const float* zpick;
  int top;
  const float* row_grad;  // nullable
  float smoothing, z_loss, inv_vocab, scale2;
  const float* rowmax;  // fp16 gradients of a scalar (else null): max |h| of each packed row
  float* unscale;       // receives the inverses of the powers of two
  float room;           // max(temperature, 1)
  int mean;
  CallState* st;
};

constexpr int kSegment = 8192;  // columns a block rescales

template <int DT>
__device__ __forceinline__ void put_dz(const RescaleArgs& a, long long off, float v) {
  if (DT == PO_F32) {
    const float h = tf32_rna(v);
    static_cast<float*>(a.e)[off] = h;
    a.lo[off] = tf32_rna(v - h);
  } else {
    typename ElemOf<DT>::T o;
    from_f32(v, o);
    static_cast<typename ElemOf<DT>::T*>(a.e)[off] = o;
  }
}

// One block: the factors of the fp16 products, and the powers of two that
// gradients of a scalar are stored by. They may lie below fp16's range until the
// caller's loss scale lifts them, a sum's also above it until the caller's
// division, and both come after the rounding here. With dZ's row at
// most 2 m in sum of magnitudes, m = coef_max times room, the mean's have
// |dH| <= 2 m max|W| / n and |dW| <= 2 m max|h|, the sum's n times as much:
// neither leaves the range by its factor (dH's takes 2 m / n away, a sum's m;
// dW's leaves half of what max|h| and a sum's n do). Where a later
// chunk of rows has a larger coef, the factors shrink, and what earlier chunks
// left is multiplied by redo_dh and redo_dw.
__device__ __forceinline__ void choose_scales(const RescaleArgs& a, float* buf) {
  CallState& st = *a.st;
  const float m = a.room * st.coef_max;
  float sh = 1.0f, sw = 1.0f;
  if (a.rowmax != nullptr) {
    float top = 0.0f;
    for (int i = threadIdx.x; i < st.count; i += blockDim.x) top = fmaxf(top, a.rowmax[i]);
    top = fmaxf(block_max(top, buf), 1e-4f) * m;
    const float n = static_cast<float>(st.counted_mean);
    if (a.mean) {
      sh = fminf(fmaxf(exp2f(floorf(log2f(n / m)) - 1.0f), 1.0f), 65536.0f);
      sw = fminf(fmaxf(exp2f(floorf(log2f(16384.0f / top))), 1.0f), 65536.0f);
    } else {
      sh = fmaxf(exp2f(floorf(log2f(1.0f / m))), 0x1p-40f);
      sw = fminf(fmaxf(exp2f(floorf(log2f(16384.0f / (top * fmaxf(n, 1.0f))))), 0x1p-40f), 65536.0f);
    }
  }
  if (threadIdx.x != 0) return;
  const bool fresh = st.store_dh == 0.0f;
  if (!fresh) sh = fminf(sh, st.store_dh), sw = fminf(sw, st.store_dw);
  st.redo_dh = fresh ? 1.0f : sh / st.store_dh;
  st.redo_dw = fresh ? 1.0f : sw / st.store_dw;
  st.store_dh = sh, st.store_dw = sw;
  const float alpha = st.alpha / f16_scale(st.coef_max);
  st.alpha_dh = alpha * sh;
  st.alpha_dw = alpha * sw;
  if (a.rowmax != nullptr) a.unscale[0] = 1.0f / sh, a.unscale[1] = 1.0f / sw;
}

// dH rows of earlier chunks brought to the factor of this one.
__global__ void __launch_bounds__(256) redo_rows_kernel(const CallState* st, const int* rowmap, int row0, __half* dh,
                                                        long long ld, int D) {
  grid_launch_next();
  grid_wait();
  const float f = st->redo_dh;
  if (f == 1.0f) return;
  const int rows = min(row0, st->count), lane = threadIdx.x & 31;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
    __half* x = dh + rowmap[r] * ld;
    for (int i = lane; i < D; i += 32) x[i] = __float2half_rn(__half2float(x[i]) * f);
  }
}

// dZ = w ((1 + 2 c lse) p - s/V - target distribution), w the row's share of
// the upstream gradient; the constant upstream factor is in the products'
// alpha, so that rounding dZ to 16 bits sees w = 1 in all but the per-row
// case. Bound by memory: 4 bytes a logit in 16-bit types.
template <int DT>
__global__ void __launch_bounds__(256) rescale_kernel(RescaleArgs a, int nseg) {
  grid_launch_next();
  grid_wait();
  __shared__ float buf[32];
  if (DT == PO_F16 && blockIdx.x == 0) choose_scales(a, buf);
  const int row = blockIdx.x / nseg;
  const int seg = blockIdx.x - row * nseg;
  const int left = a.st->count - a.row0;
  const long long base = static_cast<long long>(row) * a.e_ld;
  const int c0 = seg * kSegment;
  const int c1 = min(static_cast<long long>(c0) + kSegment, a.e_ld);
  if (row >= left) {
    if (left <= 0 || row >= (left + kRowPad - 1) / kRowPad * kRowPad) return;
    for (int c = c0 + threadIdx.x; c < c1; c += blockDim.x) put_dz<DT>(a, base + c, 0.0f);
    return;
  }
  const long long t = a.rowmap[a.row0 + row];
  const float4 stat = a.stat[row];
  const float mm = stat.x;
  const float w =
      (DT == PO_F16 ? f16_scale(a.st->coef_max) : 1.0f) * (a.row_grad != nullptr ? a.row_grad[t] / a.st->grad_max : 1.0f);
  const float coef = w * (1.0f + 2.0f * a.z_loss * stat.z);
  const float pcoef = coef * stat.y;
  const float flat = w * a.smoothing * a.inv_vocab;
  const float2* part = a.part + static_cast<long long>(row) * a.nparts;
  if (DT == PO_F32) {
#pragma unroll 2
    for (int c = c0 + threadIdx.x * 4; c < c1; c += 256 * 4) {
      const float m = part[c / a.part_cols].x;
      const float f = m == -INFINITY ? (pcoef == pcoef ? 0.0f : pcoef) : pcoef * ex2((m - mm) * a.scale2);
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.e) + base + c);
      const float x[4] = {fmaf(v.x, f, -flat), fmaf(v.y, f, -flat), fmaf(v.z, f, -flat), fmaf(v.w, f, -flat)};
      float4 h, l;
      h.x = tf32_rna(x[0]), l.x = tf32_rna(x[0] - h.x);
      h.y = tf32_rna(x[1]), l.y = tf32_rna(x[1] - h.y);
      h.z = tf32_rna(x[2]), l.z = tf32_rna(x[2] - h.z);
      h.w = tf32_rna(x[3]), l.w = tf32_rna(x[3] - h.w);
      *reinterpret_cast<float4*>(static_cast<float*>(a.e) + base + c) = h;
      *reinterpret_cast<float4*>(a.lo + base + c) = l;
    }
  } else {
    uint4 raw[4];
    float ms[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + (i * 256 + static_cast<int>(threadIdx.x)) * 8;
      if (c < c1) {
        raw[i] = *reinterpret_cast<const uint4*>(static_cast<const __half*>(a.e) + base + c);
        ms[i] = part[c / a.part_cols].x;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + (i * 256 + static_cast<int>(threadIdx.x)) * 8;
      if (c >= c1) break;
      const float m = ms[i];
      const float f = m == -INFINITY ? (pcoef == pcoef ? 0.0f : pcoef) : pcoef * ex2((m - mm) * a.scale2);
      const __half2* hv = reinterpret_cast<const __half2*>(&raw[i]);
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = __half22float2(hv[k]);
        const float x0 = fmaf(v.x, f, -flat), x1 = fmaf(v.y, f, -flat);
        o[k] = DT == PO_BF16 ? pack_bf16x2(x0, x1) : pack_f16x2(x0, x1);
      }
      *reinterpret_cast<uint4*>(static_cast<__half*>(a.e) + base + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  // The targets' columns again, with the target distribution taken off before
  // the one rounding (p from the fp32 logit).
  __syncthreads();
  for (int k = threadIdx.x; k < a.top; k += blockDim.x) {
    const int* ent = a.ent + t * a.top;
    const int c = ent[k];
    if (c < c0 || c >= c1 || (k > 0 && ent[k - 1] == c)) continue;
    float goal = 0.0f;
    if (a.q == nullptr) goal = 1.0f - a.smoothing;
    else
      for (int j = k; j < a.top && ent[j] == c; ++j) goal += a.q[t * a.top + j];
    put_dz<DT>(a, base + c, pcoef * ex2((a.zpick[t * a.top + k] - mm) * a.scale2) - flat - w * goal);
  }
}

// ------------------------------------------------------------------- join
// out[rows[row0 + r] or r][c] = alpha sum_s partial[s][r][c], in order of s.
template <int DT>
__global__ void __launch_bounds__(256) join_kernel(const float* partial, int splits, const int* splits_at, int M,
                                                   long long pld, int N, const float* alpha, const int* count, int row0,
                                                   int limit_rows, const int* rows, void* out, long long ld) {
  grid_launch_next();
  grid_wait();
  if (splits_at != nullptr) splits = *splits_at;
  if (limit_rows) M = min(M, *count - row0);
  if (splits == 1) return;  // (it wrote the output itself)
  const float al = *alpha;
  for (int r = blockIdx.x; r < M; r += gridDim.x) {
    typename ElemOf<DT>::T* o =
        static_cast<typename ElemOf<DT>::T*>(out) + (rows != nullptr ? rows[row0 + r] : r) * ld;
    for (int c = (blockIdx.y * 256 + threadIdx.x) * 4; c < N; c += gridDim.y * 1024) {
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(partial + (static_cast<long long>(k) * M + r) * pld + c);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      const float x[4] = {s.x * al, s.y * al, s.z * al, s.w * al};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < N) from_f32(x[i], o[c + i]);
    }
  }
}

// Zeroes a rows x cols matrix (no counted row can reach it).
template <int DT>
__global__ void zero_kernel(void* out, long long ld, long long rows, long long cols) {
  typename ElemOf<DT>::T z;
  from_f32(0.0f, z);
  for (long long r = blockIdx.x; r < rows; r += gridDim.x)
    for (long long c = threadIdx.x; c < cols; c += blockDim.x)
      static_cast<typename ElemOf<DT>::T*>(out)[r * ld + c] = z;
}

// ------------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// rows x cols matrix of `dtype`, pitch ld; boxes of box_cols x box_rows, zeros outside.
int encode(CUtensorMap* map, const void* ptr, int dtype, long long rows, long long cols, long long ld, int box_cols,
           int box_rows, bool mn) {
  auto fn = encode_fn();
  if (fn == nullptr) return set_error(PO_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const int es = dtype_size(dtype);
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), 1};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * es), static_cast<cuuint64_t>(ld * es * rows)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType t = dtype == PO_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : dtype == PO_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                   : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUtensorMapSwizzle swz =
      mn && es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B;
  const CUresult r = fn(map, t, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PO_OK : set_error(PO_ERR_CUDA, "linear_loss: cuTensorMapEncodeTiled failed");
}

// One operand of a product: hi (and lo) matrices, stored K-major [MN][K] or
// MN-major [K][MN].
struct HeadOperand {
  const void* p[2];
  int dtype;
  long long rows, cols, ld;
  bool kmajor;
};

int encode_operand(CUtensorMap map[2], const HeadOperand& o) {
  const int es = dtype_size(o.dtype);
  const int w = 128 / es;
  for (int i = 0; i < 2; ++i) {
    const void* p = o.p[i];
    if (p == nullptr) {  // no low half: never read
      map[i] = map[0];
      continue;
    }
    // K-major: 128 bytes of K x 128 rows; MN-major: 128 bytes of MN x a stage's rows of K.
    const int r = o.kmajor ? encode(&map[i], p, o.dtype, o.rows, o.cols, o.ld, w, 128, false)
                           : encode(&map[i], p, o.dtype, o.rows, o.cols, o.ld, w, es == 4 ? w : 2 * w, true);
    if (r) return r;
  }
  return PO_OK;
}

// Splits of K for a store product.
int choose_splits(long long tiles, int nkb, long long M, long long N) {
  const int pairs = sm_count() / 2;
  if (tiles > 16 * pairs) return 1;  // (a last wave weighs little)
  const float values = static_cast<float>(M) * static_cast<float>(N);
  int best = 1;
  float best_cost = INFINITY;
  for (int s = 1; s <= pairs && s <= (nkb + 3) / 4; ++s) {
    const float cost = split_cost(s, static_cast<int>(tiles), nkb, values, pairs);
    if (cost < best_cost * 0.98f) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}

// Sizes and places of one call.
struct Plan {
  long long T, D, V, top;
  int dtype, es;
  bool f32, soft, grads, want_dh, want_dw;
  bool few;           // up to kFewRows rows: logits on the CUDA cores
  int part_cols;      // columns a partial statistic covers
  long long chunk;    // rows a pass of the products takes
  int nchunks;
  long long rows_alloc;
  long long ldp;      // pitch of packed H and staged W
  bool stage_w;
  int nparts;
  long long e_ld;
  int bk;
  float* rowmax;
  int splits_dh, splits_dw;
  int dh_blocks, split_units;  // dH's splits are chosen on the device (0: they are not)
  bool dw_acc;
  // workspace
  CallState* st;
  unsigned int* sched;
  int* rowmap;
  int* status;
  int* ent;
  float* q;
  float* qlogq;
  float* zpick;
  float4* stat;
  float2* part;
  float* zsum;
  void* packed;
  float* packed_lo;
  void* w;
  float* w_lo;
  void* e;
  float* e_lo;
  float* partial;
  float* dw_accum;
  size_t bytes;
};

// Rows up to which the CUDA cores make the logits. A whole call without
// gradients, CUDA cores against tensor cores, us: bf16, 50257 x 768, 1 row 25 /
// 37, 4 rows 33 / 33, fp16 8 rows 53 / 34; bf16, 128256 x 4096, 2 rows 205 /
// 257, 4 rows 258 / 260, 8 rows 485 / 283; fp32 (where the tensor cores need W
// split into pairs first), 50257 x 768, 8 rows 68 / 203.
int few_rows(int dtype) { return dtype == PO_F32 ? kFewRows : 2; }

// Rows a pass keeps in the workspace by default: as many as leave 2 GiB of
// exponentials (8191 rows of 128 thousand columns in 16 bits).
constexpr long long kDefaultChunkBytes = 2LL << 30;

int make_plan(Plan& p, const void* weight, long long w_ld, int dtype, long long T, long long D, long long V,
              long long top, bool soft, bool few, bool want_dh, bool want_dw, long long chunk_rows, void* ws,
              size_t ws_bytes) {
  memset(&p, 0, sizeof(p));
  p.T = T, p.D = D, p.V = V, p.top = top, p.dtype = dtype, p.es = dtype_size(dtype);
  p.f32 = dtype == PO_F32;
  p.soft = soft;
  p.want_dh = want_dh, p.want_dw = want_dw, p.grads = want_dh || want_dw;
  p.ldp = round_up(D, 64);
  p.few = few;
  // The few-rows kernel takes W as it is; the tensor cores need pitches that
  // TMA takes, and fp32 as tf32 pairs.
  p.stage_w = (!p.few || want_dh) && (p.f32 || reinterpret_cast<uintptr_t>(weight) % 16 != 0 || (w_ld * p.es) % 16 != 0);
  p.part_cols = p.few ? kFewPartCols : kPartCols;
  p.e_ld = round_up(V, 256);
  p.nparts = static_cast<int>(p.e_ld / p.part_cols);
  p.bk = p.f32 ? 32 : 128;
  long long most = chunk_rows;
  if (most <= 0) {
    // Without gradients a row leaves 8 bytes per 256 columns.
    const long long per_row = p.grads ? p.e_ld * (p.f32 ? 8 : 2) : static_cast<long long>(p.nparts) * 8;
    most = kDefaultChunkBytes / per_row;
  }
  most = most / 256 * 256;
  if (most < 256) most = 256;
  p.nchunks = static_cast<int>((T + most - 1) / most);
  p.chunk = p.nchunks == 1 ? T : round_up((T + p.nchunks - 1) / p.nchunks, 256);
  p.rows_alloc = round_up(T, kRowPad);
  const long long mt = (p.chunk + 255) / 256, nd = (D + 255) / 256, nv = (V + 255) / 256;
  // K blocks in units of a 16-bit one's time (an fp32 block issues 1.5 times as much).
  const auto blocks = [&](long long k) { return p.f32 ? cdiv(3LL * cdiv(k, p.bk), 2) : cdiv(k, p.bk); };
  p.splits_dh = want_dh ? choose_splits(mt * nd, blocks(V), p.chunk, D) : 1;
  // Fewer rows may count, and fewer tiles then take more splits: the finishing
  // kernel chooses, within 256 KB a tile and split and two units a pair of SMs.
  if (want_dh && mt > 1 && mt * nd <= 16 * (sm_count() / 2)) {
    p.dh_blocks = blocks(V);
    const long long units = mt * nd * p.splits_dh;
    p.split_units = static_cast<int>(units > 2 * (sm_count() / 2) ? units : 2 * (sm_count() / 2));
  }
  p.dw_acc = want_dw && p.nchunks > 1;
  p.splits_dw = want_dw && !p.dw_acc ? choose_splits(nv * nd, blocks(p.chunk), V, D) : 1;

  Arena ar(ws, ws_bytes);
  auto i32 = [&](long long n) { return static_cast<int*>(ar.take(static_cast<size_t>(n) * 4)); };
  auto f32 = [&](long long n) { return static_cast<float*>(ar.take(static_cast<size_t>(n) * 4)); };
  p.st = static_cast<CallState*>(ar.take(sizeof(CallState)));
  p.sched = static_cast<unsigned int*>(ar.take(8));
  p.rowmap = i32(T);
  if (dtype == PO_F16) p.rowmax = f32(T);
  p.ent = i32(T * top);
  p.zpick = f32(T * top);
  if (soft) {
    p.status = i32(T);
    p.q = f32(T * top);
    p.qlogq = f32(T);
  }
  p.stat = static_cast<float4*>(ar.take(static_cast<size_t>(p.chunk) * 16));
  p.part = static_cast<float2*>(ar.take(static_cast<size_t>(p.chunk) * p.nparts * 8));
  p.zsum = f32(soft ? 1 : p.chunk * p.nparts);
  p.packed = ar.take(static_cast<size_t>(p.rows_alloc) * p.ldp * p.es);
  if (p.f32) p.packed_lo = f32(p.rows_alloc * p.ldp);
  if (p.stage_w) {
    p.w = ar.take(static_cast<size_t>(V) * p.ldp * p.es);
    if (p.f32) p.w_lo = f32(V * p.ldp);
  }
  if (p.grads) {
    const long long rows = round_up(p.chunk, kRowPad);
    p.e = ar.take(static_cast<size_t>(rows) * p.e_ld * p.es);
    if (p.f32) p.e_lo = f32(rows * p.e_ld);
    const long long pld = round_up(D, 256);
    long long partial = 0;
    if (p.split_units > 0) partial = static_cast<long long>(p.split_units) * (256 * 256);
    else if (p.splits_dh > 1) partial = p.splits_dh * p.chunk * pld;
    if (p.splits_dw > 1 && p.splits_dw * V * pld > partial) partial = p.splits_dw * V * pld;
    if (partial > 0) p.partial = f32(partial);
    if (p.dw_acc && !p.f32) p.dw_accum = f32(V * round_up(D, 8));
  }
  p.bytes = ar.used;
  return ar.overflow() ? set_error(PO_ERR_WORKSPACE, "linear_loss: workspace too small") : PO_OK;
}

int join(int dtype, const float* alpha, const float* partial, int splits, const int* splits_at, int M, long long pld,
         int N, const Plan& p, int row0, bool limit_rows, const int* rows, void* out, long long ld, cudaStream_t s) {
  // Blocks that fit at once: the launch costs little where there is one split.
  const dim3 grid(M < 8 * sm_count() ? M : 8 * sm_count(), N > 4096 ? 4 : 1);
  const auto kern = dtype == PO_F32 ? join_kernel<PO_F32> : dtype == PO_BF16 ? join_kernel<PO_BF16> : join_kernel<PO_F16>;
  return launch_next(false, kern, grid, 256, 0, s, "linear_loss join", partial, splits, splits_at, M, pld, N, alpha,
                     &p.st->count, row0, limit_rows, rows, out, ld);
}

int run_head(const Plan& p, int product, HeadParams& P, const HeadOperand& A, const HeadOperand& B, int splits,
             cudaStream_t s) {
  int r;
  if ((r = encode_operand(P.mapA, A))) return r;
  if ((r = encode_operand(P.mapB, B))) return r;
  P.count = &p.st->count;
  P.sched = p.sched;
  P.err = device_error_word();
  if (P.err == nullptr) return set_error(PO_ERR_CUDA, "device error word unavailable");
  P.fmt = p.f32 ? 2u : (p.dtype == PO_BF16 ? 1u : 0u);
  P.splits = splits;
  P.tiles_n = cdiv(P.N, 256);
  const int tiles_m = cdiv(P.M, 256);
  // (splits chosen on the device may make more units of fewer tiles: as many as their workspace holds)
  long long tiles = static_cast<long long>(tiles_m) * P.tiles_n * splits;
  if (P.splits_at != nullptr && tiles < p.split_units) tiles = p.split_units;
  if (tiles > INT_MAX / 2) return set_error(PO_ERR_ARG, "linear_loss: too many tiles");
  return p.f32 ? dispatch_head<KIND_TF32>(product, P, static_cast<int>(tiles), s)
               : dispatch_head<KIND_BF16>(product, P, static_cast<int>(tiles), s);
}

// K blocks summed inside the tensor core's accumulator, which truncates. 16-bit
// operands (blocks of 128 of K): a mean loss is off by 2e-7 with 2 and 4e-7 with
// 4 blocks; 2047 x 128256 x 4096 takes 1.56 and 1.45 ms, 8191 x 32000 x 2048
// with gradients 753 and 708 us, 8 blocks save nothing more. 16-bit gradients
// round to 2^-9: 2048 of K. fp32 (blocks of 32 of K), 500 x 50257 x 768: with 1
// and 2 blocks in the logits the loss is off by 1.1e-7 and 2.9e-7 and the
// gradients by 4e-7 and 5e-7, and the logits take 214 and 196 us of 700 and 680;
// few confident rows, whose gradients are small differences, need the former.
constexpr int kChunkStats16 = 4, kChunkStats32 = 1, kChunkGrad16 = 16, kChunkGrad32 = 4;

bool vec32(const void* p, long long ld, int es) {
  return reinterpret_cast<uintptr_t>(p) % 32 == 0 && (ld * es) % 32 == 0;
}

}  // namespace
}  // namespace po

using namespace po;

extern "C" size_t po_linear_loss_workspace_bytes(const void* weight, long long w_ld, int dtype, long long tokens,
                                                 long long dim, long long vocab, long long top, int want_dhidden,
                                                 int want_dweight, long long chunk_rows) {
  if (tokens <= 0 || dim <= 0 || vocab <= 0 || top <= 0 || dtype_size(dtype) == 0) return 0;
  Plan p;
  // Enough for both kinds of targets, and for hidden rows on any boundary.
  size_t best = 0;
  for (int soft = 0; soft < 2; ++soft)
    for (int few = 0; few < (tokens <= few_rows(dtype) ? 2 : 1); ++few) {
      make_plan(p, weight, w_ld, dtype, tokens, dim, vocab, top, soft != 0, few != 0, want_dhidden != 0,
                want_dweight != 0, chunk_rows, nullptr, 0);
      if (p.bytes > best) best = p.bytes;
    }
  return best + 256;
}

extern "C" int po_linear_loss(const void* hidden, long long h_ld, const void* weight, long long w_ld, int dtype,
                              long long tokens, long long dim, long long vocab, const long long* index,
                              long long index_ld, const void* teacher, long long teacher_ld, int teacher_dtype,
                              long long top, long long ignore_index, float smoothing, float z_loss, float temperature,
                              int mean, const float* row_grad, float* loss_rows, float* loss, void* dhidden,
                              long long dh_ld, void* dweight, long long dw_ld, long long chunk_rows, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (dtype != PO_F32 && dtype != PO_BF16 && dtype != PO_F16)
    return set_error(PO_ERR_ARG, "linear_loss: dtype must be fp32, bf16 or fp16");
  if (tokens < 0 || dim <= 0 || vocab <= 0) return set_error(PO_ERR_ARG, "linear_loss: bad size");
  if (tokens > (1 << 26) || dim > (1 << 24) || vocab > (1 << 28))
    return set_error(PO_ERR_ARG, "linear_loss: size too large");
  // An empty call reads no targets, and its teacher may have no address: it may be of either kind.
  const bool soft = teacher != nullptr, hard = !soft && tokens > 0;
  if (top < 1 || top > kMaxTop || (hard && top != 1))
    return set_error(PO_ERR_ARG, "linear_loss: top must be 1 to 1024 (1 without a teacher)");
  if (soft && teacher_dtype != PO_F32 && teacher_dtype != PO_BF16 && teacher_dtype != PO_F16)
    return set_error(PO_ERR_ARG, "linear_loss: teacher dtype must be fp32, bf16 or fp16");
  if (!temperature_ok(temperature) || (hard && temperature != 1.0f))
    return set_error(PO_ERR_ARG, "linear_loss: temperature must be 2^-60 to 2^60 (1 without a teacher)");
  if (!(smoothing >= 0.0f && smoothing <= 1.0f) || !std::isfinite(z_loss) || (soft && (smoothing != 0.0f || z_loss != 0.0f)))
    return set_error(PO_ERR_ARG, "linear_loss: smoothing must be in [0, 1] and z_loss finite (both 0 with a teacher)");
  const bool scaled = mean == PO_MEAN_SCALED || mean == PO_SUM_SCALED;
  if (row_grad != nullptr && (mean || (dhidden == nullptr && dweight == nullptr)))
    return set_error(PO_ERR_ARG, "linear_loss: row_grad goes with gradients of the sum");
  if (h_ld < dim || w_ld < dim || (tokens > 1 && (index_ld < top || (soft && teacher_ld < top))) ||
      (dhidden != nullptr && dh_ld < dim) || (dweight != nullptr && dw_ld < dim))
    return set_error(PO_ERR_ARG, "linear_loss: a pitch is smaller than its row");
  if (weight == nullptr || (tokens > 0 && (hidden == nullptr || index == nullptr || loss_rows == nullptr)))
    return set_error(PO_ERR_ARG, "linear_loss: null operand");
  if (mean == PO_SUM_SCALED) mean = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count();
  if (tokens == 0) {
    if (loss != nullptr)
      if (int r = check_cuda(cudaMemsetAsync(loss, 0, 4, s), "linear_loss")) return r;
    if (dweight != nullptr) {
      if (dtype == PO_F32) zero_kernel<PO_F32><<<8 * sms, 256, 0, s>>>(dweight, dw_ld, vocab, dim);
      else zero_kernel<PO_BF16><<<8 * sms, 256, 0, s>>>(dweight, dw_ld, vocab, dim);
      return check_cuda(cudaGetLastError(), "linear_loss zero");
    }
    return PO_OK;
  }
  if (workspace == nullptr) return set_error(PO_ERR_WORKSPACE, "linear_loss: workspace too small");
  Plan p;
  const auto aligned = [&](const void* x, long long ld) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * dtype_size(dtype) % 16 == 0;
  };
  const bool few = tokens <= few_rows(dtype) && aligned(hidden, h_ld) && aligned(weight, w_ld);
  int r = make_plan(p, weight, w_ld, dtype, tokens, dim, vocab, top, soft, few, dhidden != nullptr, dweight != nullptr,
                    chunk_rows, workspace, workspace_bytes);
  if (r) return r;
  const int T = static_cast<int>(tokens), D = static_cast<int>(dim), V = static_cast<int>(vocab);
  const Targets tg{index, index_ld, teacher, teacher_ld, teacher_dtype, static_cast<int>(top), ignore_index};

  bool first = true;
  if (soft) {
    int width = 2;
    while (width < top) width <<= 1;
    const int threads = width < 64 ? 32 : (width > 256 ? 128 : width / 2);
    if ((r = launch_next(first, teacher_targets_kernel, T, threads, width * 8, s, "linear_loss targets", tg, vocab,
                         1.0f / temperature, width, p.status, p.ent, p.q, p.qlogq)))
      return r;
    first = false;
  }
  PackArgs pa{};
  pa.hidden = hidden, pa.h_ld = h_ld, pa.T = tokens, pa.D = D, pa.ldp = static_cast<int>(p.ldp);
  pa.vec = D * p.es % 16 == 0 && reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && h_ld * p.es % 16 == 0;
  pa.tg = tg, pa.V = vocab, pa.status = p.status, pa.ent = p.ent, pa.rowmap = p.rowmap;
  pa.packed = p.packed, pa.packed_lo = p.packed_lo;
  pa.dhidden = dhidden, pa.dh_ld = dh_ld, pa.loss_rows = loss_rows, pa.st = p.st, pa.sched = p.sched;
  pa.alpha = temperature, pa.mean = mean, pa.has_row_grad = row_grad != nullptr;
  float* unscale = scaled && p.grads ? loss_rows + tokens : nullptr;
  pa.unscale = unscale, pa.rowmax = unscale != nullptr && dtype == PO_F16 ? p.rowmax : nullptr;
  if (row_grad != nullptr) {
    if ((r = launch_next(first, grad_max_kernel, 1, 1024, 0, s, "linear_loss grad_max", pa, row_grad))) return r;
    first = false;
  }
  const int groups = cdiv(T, 2048 * kPackWarps), pblocks = cdiv(T, groups * kPackWarps);
  const auto pack = dtype == PO_F32 ? pack_kernel<PO_F32> : dtype == PO_BF16 ? pack_kernel<PO_BF16> : pack_kernel<PO_F16>;
  if ((r = launch_next(first, pack, pblocks, 32 * kPackWarps, 0, s, "linear_loss pack", pa, groups))) return r;

  const void* w = weight;
  long long wld = w_ld;
  if (p.stage_w) {
    const int vec = p.f32 && dim % 4 == 0 && w_ld % 4 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0;
    if ((r = launch_next(false, p.f32 ? stage_weight_kernel<PO_F32> : stage_weight_kernel<PO_BF16>, 8 * sms, 256, 0, s,
                         "linear_loss stage", weight, w_ld, vocab, D, static_cast<int>(p.ldp), p.w, p.w_lo, vec)))
      return r;
    w = p.w;
    wld = p.ldp;
  }

  for (int c = 0; c < p.nchunks; ++c) {
    const long long row0 = c * p.chunk;
    const int rows = static_cast<int>(tokens - row0 < p.chunk ? tokens - row0 : p.chunk);
    const size_t hoff = static_cast<size_t>(row0) * p.ldp;
    const void* hp = static_cast<const char*>(p.packed) + hoff * p.es;
    const float* hlo = p.f32 ? p.packed_lo + hoff : nullptr;
    const long long krows = round_up(rows, kRowPad);
    const HeadOperand Hk{{hp, hlo}, dtype, rows, dim, p.ldp, true};
    const HeadOperand Wk{{w, p.w_lo}, dtype, vocab, dim, wld, true};
    FinishArgs fa{};
    fa.part = p.part, fa.zsum = smoothing != 0.0f ? p.zsum : nullptr, fa.nparts = p.nparts, fa.row0 = static_cast<int>(row0);
    fa.rowmap = p.rowmap, fa.zpick = p.zpick, fa.ent = p.ent, fa.q = soft ? p.q : nullptr, fa.qlogq = p.qlogq;
    fa.top = static_cast<int>(top), fa.smoothing = smoothing, fa.z_loss = z_loss;
    fa.temperature = temperature, fa.scale2 = kLog2e / temperature;
    fa.inv_vocab = 1.0f / static_cast<float>(vocab), fa.stat = p.stat, fa.loss_rows = loss_rows, fa.loss = loss;
    fa.T = tokens, fa.mean = mean, fa.final_launch = c == p.nchunks - 1, fa.st = p.st;
    if (p.want_dw) {
      fa.packed = static_cast<uint4*>(p.packed) + hoff * p.es / 16;
      fa.packed_lo = p.f32 ? reinterpret_cast<uint4*>(p.packed_lo + hoff) : nullptr;
      fa.row_words = static_cast<int>(p.ldp * p.es / 16);
    }
    fa.rows = rows;
    if (p.split_units > 0) fa.split = {p.dh_blocks, cdiv(D, 256), D, sm_count() / 2, p.split_units};
    if (p.few) {
      FewParams P{};
      P.h = hidden, P.h_ld = h_ld, P.w = weight, P.w_ld = w_ld, P.D = D, P.V = V;
      P.scale2 = kLog2e / temperature, P.part = p.part, P.zsum = smoothing != 0.0f ? p.zsum : nullptr;
      P.e = p.e, P.e_ld = p.e_ld, P.zpick = p.zpick;
      P.finish = fa;
      if ((r = launch_few_rows(P, dtype, T, s))) return r;
    } else {
      HeadParams P;
      memset(&P, 0, sizeof(P));
      P.M = rows, P.N = V, P.K = D, P.limit = LIMIT_M, P.row0 = static_cast<int>(row0);
      // All row tiles of a vocabulary tile run together (W is read once) as
      // long as their panels of H take at most 48 MB of L2.
      const int mt = cdiv(rows, 256);
      const long long panel = 256LL * p.ldp * p.es * (p.f32 ? 2 : 1);
      const int fit = static_cast<int>((48LL << 20) / panel > 1 ? (48LL << 20) / panel : 1);
      P.band = cdiv(mt, cdiv(mt, fit));
      P.chunk = p.f32 ? kChunkStats32 : kChunkStats16;
      P.scale2 = kLog2e / temperature;
      P.part = p.part, P.nparts = p.nparts, P.zsum = smoothing != 0.0f ? p.zsum : nullptr;
      P.e = p.e, P.e_ld = p.e_ld, P.rowmap = p.rowmap, P.ent = p.ent, P.top = static_cast<int>(top), P.zpick = p.zpick;
      if ((r = run_head(p, HEAD_LOGITS, P, Hk, Wk, 1, s))) return r;
    }
    if (!p.few && (r = launch_next(false, finish_kernel, cdiv(p.want_dw ? krows : rows, kFinishWarps), 32 * kFinishWarps,
                                   0, s, "linear_loss finish", fa)))
      return r;
    if (!p.grads) continue;

    RescaleArgs ra{};
    ra.e = p.e, ra.lo = p.e_lo, ra.e_ld = p.e_ld, ra.V = vocab, ra.part = p.part, ra.nparts = p.nparts, ra.part_cols = p.part_cols, ra.stat = p.stat;
    ra.row0 = static_cast<int>(row0), ra.rows = rows, ra.rowmap = p.rowmap, ra.ent = p.ent, ra.q = soft ? p.q : nullptr;
    ra.scale2 = kLog2e / temperature, ra.zpick = p.zpick, ra.top = static_cast<int>(top), ra.row_grad = row_grad, ra.smoothing = smoothing;
    ra.z_loss = z_loss, ra.inv_vocab = 1.0f / static_cast<float>(vocab), ra.st = p.st;
    ra.rowmax = pa.rowmax, ra.unscale = unscale, ra.room = fmaxf(temperature, 1.0f), ra.mean = mean;
    const int nseg = cdiv(p.e_ld, kSegment);
    const long long rblocks = krows * nseg;
    if (rblocks > INT_MAX) return set_error(PO_ERR_ARG, "linear_loss: chunk too large");
    const auto rescale =
        dtype == PO_F32 ? rescale_kernel<PO_F32> : dtype == PO_BF16 ? rescale_kernel<PO_BF16> : rescale_kernel<PO_F16>;
    if ((r = launch_next(false, rescale, static_cast<int>(rblocks), 256, 0, s, "linear_loss rescale", ra, nseg))) return r;

    const long long pld = round_up(dim, 256);
    const bool redo = pa.rowmax != nullptr && z_loss != 0.0f && c > 0;  // (without a z-loss the factors stay)
    if (redo && p.want_dh &&
        (r = launch_next(false, redo_rows_kernel, sms, 256, 0, s, "linear_loss redo", p.st, p.rowmap,
                         static_cast<int>(row0), static_cast<__half*>(dhidden), dh_ld, D)))
      return r;
    if (p.want_dh) {
      HeadParams P;
      memset(&P, 0, sizeof(P));
      P.M = rows, P.N = D, P.K = V, P.limit = LIMIT_M, P.row0 = static_cast<int>(row0), P.band = 8;
      P.chunk = p.f32 ? kChunkGrad32 : kChunkGrad16;
      P.alpha = &p.st->alpha_dh, P.out = dhidden, P.out_ld = dh_ld, P.out_dtype = dtype, P.vec = vec32(dhidden, dh_ld, p.es);
      P.out_rows = p.rowmap, P.partial = p.partial, P.part_ld = pld;
      const HeadOperand A{{p.e, p.e_lo}, dtype, rows, vocab, p.e_ld, true};
      const HeadOperand B{{w, p.w_lo}, dtype, vocab, dim, wld, false};
      P.splits_at = p.split_units > 0 ? &p.st->splits : nullptr;
      if ((r = run_head(p, HEAD_DHIDDEN, P, A, B, p.splits_dh, s))) return r;
      if ((p.splits_dh > 1 || P.splits_at != nullptr) &&
          (r = join(dtype, P.alpha, p.partial, p.splits_dh, P.splits_at, rows, pld, D, p, static_cast<int>(row0), true, p.rowmap, dhidden, dh_ld, s)))
        return r;
    }
    if (p.want_dw) {
      HeadParams P;
      memset(&P, 0, sizeof(P));
      P.M = V, P.N = D, P.K = rows, P.limit = LIMIT_K, P.row0 = static_cast<int>(row0), P.band = 8;
      P.chunk = p.f32 ? kChunkGrad32 : kChunkGrad16;
      P.alpha = &p.st->alpha_dw, P.partial = p.partial, P.part_ld = pld;
      const bool to_acc = p.dw_acc && !p.f32;  // fp32 gradients add up in place
      const bool last = c == p.nchunks - 1;
      float* acc = to_acc ? p.dw_accum : static_cast<float*>(dweight);
      const long long acc_ld = to_acc ? round_up(dim, 8) : dw_ld;
      P.cin = p.dw_acc && c > 0 ? acc : nullptr;
      P.cin_ld = acc_ld;
      P.cin_scale = redo ? &p.st->redo_dw : nullptr;
      const bool mid = to_acc && !last;
      P.out = mid ? static_cast<void*>(acc) : dweight;
      P.out_ld = mid ? acc_ld : dw_ld;
      P.out_dtype = mid ? PO_F32 : dtype;
      P.vec = vec32(P.out, P.out_ld, dtype_size(P.out_dtype)) && (P.cin == nullptr || vec32(P.cin, acc_ld, 4));
      // Rows past the counted ones are zero up to a K block in both operands.
      const HeadOperand A{{p.e, p.e_lo}, dtype, krows, vocab, p.e_ld, false};
      const HeadOperand B{{hp, hlo}, dtype, p.rows_alloc - row0 < krows ? p.rows_alloc - row0 : krows, dim, p.ldp, false};
      if ((r = run_head(p, HEAD_DWEIGHT, P, A, B, p.splits_dw, s))) return r;
      if (p.splits_dw > 1 && (r = join(dtype, P.alpha, p.partial, p.splits_dw, nullptr, V, pld, D, p, 0, false, nullptr, dweight, dw_ld, s)))
        return r;
    }
  }
  return PO_OK;
}
