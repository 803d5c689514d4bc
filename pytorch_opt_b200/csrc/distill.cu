// Divergence of student logits from a teacher's top logits, with its gradient
// (po_distill_logits), and the scaling of gradients by a device scalar.
//
//   q = softmax(teacher / a),  l = a^2 sum_k q_k (log q_k + lse(z/a) - z_k/a),
//   dz = a (softmax(z / a) - q scattered)
//
// Bound by memory: each logit is read once and each gradient written once (4
// bytes a logit in 16-bit types). A row's sum has to be known before its first
// gradient is written, so a row stays on the chip in between: a cluster of up
// to 8 CTAs shares one row, each CTA keeps its segment in shared memory, and
// the CTAs exchange their (max, sum) through distributed shared memory. Short
// segments keep several CTAs on an SM, so that one loads while another writes;
// a single long row is spread over 8 SMs.
#include <climits>
#include <cmath>

#include "head_gemm.cuh"
#include "losses.cuh"

namespace po {
namespace {

struct DistillState {
  int count;  // rows that the mean divides by
  unsigned int done;
};

struct DistillArgs {
  const void* z;
  long long ld;
  void* dz;  // nullable
  long long dz_ld;
  long long T;
  int V;
  const long long* index;
  long long index_ld;
  const void* teacher;
  long long teacher_ld;
  int teacher_dtype;
  int top;
  float temperature;
  int mean;
  const float* row_grad;
  float* loss_rows;
  float* loss;
  DistillState* st;
  int seg;     // elements a CTA takes
  int cached;  // the segment stays in shared memory
};

// Whether the row has an entry with mass; bad indices are found here too.
__device__ __forceinline__ int entry_status(const DistillArgs& a, long long t, int k, long long& x, float& l) {
  x = a.index[t * a.index_ld + k];
  l = -INFINITY;
  if (x >= a.V) return ROW_BAD;
  if (x < 0) return ROW_IGNORED;
  l = load_as_f32(a.teacher, a.teacher_dtype, t * a.teacher_ld + k);
  return l > -INFINITY || isnan(l) ? ROW_COUNTED : ROW_IGNORED;
}

// Rows that the mean divides by (counted ones and those with a bad index).
__global__ void __launch_bounds__(256) count_rows_kernel(DistillArgs a) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  int n = 0;
  for (long long t = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); t < a.T; t += warps) {
    bool any = false;
    for (int k = lane; k < a.top; k += 32) {
      long long x;
      float l;
      any |= entry_status(a, t, k, x, l) != ROW_IGNORED;
    }
    n += __any_sync(0xffffffffu, any) ? 1 : 0;
  }
  if (lane == 0 && n > 0) atomicAdd(&a.st->count, n);
}

__device__ __forceinline__ float4 ld_cluster_f4(const float4* p, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(mapa_shared(smem_u32(p), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// (m, s) <- (m, s) joined with 2^(scale2 x); the sum is kept relative to the
// maximum, which is subtracted before the scaling: z - m is exact where it matters.
template <int N>
__device__ __forceinline__ void online_add(const float (&x)[N], float scale2, float& m, float& s) {
  float c = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) c = fmaxf(c, x[i]);
  if (c > m) {
    s *= ex2((m - c) * scale2);
    m = c;
  }
  const float off = m == -INFINITY ? 0.0f : m;
  float add = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) add += ex2((x[i] - off) * scale2);
  s += add;
}

constexpr int kDistillThreads = 256;

template <int DT, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads) distill_kernel(DistillArgs a) {
  using T = typename ElemOf<DT>::T;
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ float buf[32];
  __shared__ double dbuf[32];
  __shared__ __align__(16) float4 s_share;
  __shared__ int s_last;
  const uint32_t cs = cluster_nctarank(), rank = cluster_ctarank();
  const long long t = blockIdx.x / cs;
  int* si = reinterpret_cast<int*>(sm);            // entries' indices (-1: none)
  float* sq = reinterpret_cast<float*>(si + a.top);  // q
  float* sz = sq + a.top;                            // logits at the entries
  T* cache = reinterpret_cast<T*>(sm + (static_cast<size_t>(a.top) * 12 + 15) / 16 * 16);
  const float scale2 = kLog2e / a.temperature;

  const T* z = static_cast<const T*>(a.z) + t * a.ld;
  const int s0 = min(static_cast<long long>(rank) * a.seg, static_cast<long long>(a.V));
  const int s1 = min(static_cast<long long>(s0) + a.seg, static_cast<long long>(a.V));
  // Vectors lie on 16-byte boundaries of the logits; the first holds `mis`
  // elements that belong to someone else (never read).
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(z + s0) / sizeof(T)) % VEC);
  const int nvec = (s1 - s0 + mis + VEC - 1) / VEC;

  // Teacher's distribution (every CTA of the row for itself).
  float tm = -INFINITY;
  bool bad = false, mass = false;
  for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
    long long x;
    float l;
    const int e = entry_status(a, t, k, x, l);
    bad |= e == ROW_BAD;
    mass |= e == ROW_COUNTED;
    const bool there = x >= 0 && x < a.V;
    si[k] = there ? static_cast<int>(x) : -1;
    l = there ? l / a.temperature : -INFINITY;
    sq[k] = l;
    sz[k] = there ? to_f32(z[x]) : 0.0f;
    tm = fmaxf(tm, l);
  }
  bad = __syncthreads_or(bad);
  mass = __syncthreads_or(mass);

  float m = -INFINITY, s = 0.0f;
  float qlogq = 0.0f;
  if (mass && !bad) {
    // Segment: running maximum and sum, four vectors in flight a thread.
    const T* z0 = z + s0 - mis;
    for (int j0 = threadIdx.x; j0 < nvec; j0 += 4 * kDistillThreads) {
      uint4 raw[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * kDistillThreads;
        if (j >= nvec) continue;
        if ((j > 0 || mis == 0) && (j + 1) * VEC <= s1 - s0 + mis) {
          raw[u] = __ldcs(reinterpret_cast<const uint4*>(z0) + j);
        } else {
          T* o = reinterpret_cast<T*>(&raw[u]);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int c = j * VEC + i;
            from_f32(-INFINITY, o[i]);
            if (c >= mis && c < s1 - s0 + mis) o[i] = z0[c];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u * kDistillThreads;
        if (j >= nvec) continue;
        float x[VEC];
        const T* o = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = to_f32(o[i]);
        online_add(x, scale2, m, s);
        if (GRAD && a.cached) reinterpret_cast<uint4*>(cache)[j] = raw[u];
      }
    }
    const float mm = block_max(m, buf);
    s = block_sum(m == -INFINITY ? s : s * ex2((m - mm) * scale2), buf);
    m = mm;
    // q and sum q log q
    tm = block_max(tm, buf);
    float sum = 0.0f;
    for (int k = threadIdx.x; k < a.top; k += kDistillThreads)
      if (si[k] >= 0) sum += expf(sq[k] - tm);
    sum = block_sum(sum, buf);
    const float logsum = logf(sum);
    for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
      float q = 0.0f;
      if (si[k] >= 0) {
        q = expf(sq[k] - tm) / sum;
        if (q != 0.0f) qlogq += q * (sq[k] - tm - logsum);
      }
      sq[k] = q;
    }
    qlogq = block_sum(qlogq, buf);
    // Join the row's CTAs, each in rank order.
    if (cs > 1) {
      if (threadIdx.x == 0) s_share = make_float4(m, s, 0.0f, 0.0f);
      cluster_sync();
      float gm = -INFINITY, gs = 0.0f;
      float4 v[8];
#pragma unroll
      for (uint32_t r = 0; r < 8; ++r)
        if (r < cs) {
          v[r] = ld_cluster_f4(&s_share, r);
          gm = fmaxf(gm, v[r].x);
        }
#pragma unroll
      for (uint32_t r = 0; r < 8; ++r)
        if (r < cs) gs += v[r].x == -INFINITY ? v[r].y : v[r].y * ex2((v[r].x - gm) * scale2);
      m = gm;
      s = gs;
    }
  }
  const float logs = logf(s);  // log sum exp(z / a) = m / a + logs

  if (rank == 0) {
    float c = 0.0f;
    if (mass && !bad)
      for (int k = threadIdx.x; k < a.top; k += kDistillThreads)
        if (sq[k] != 0.0f) c += sq[k] * ((m - sz[k]) / a.temperature + logs);
    c = block_sum(c, buf);
    if (threadIdx.x == 0) {
      float loss = 0.0f;
      if (bad) loss = NAN;
      else if (mass) loss = a.temperature * a.temperature * (qlogq + c);
      a.loss_rows[t] = loss;
    }
  }

  if (GRAD) {
    T* out = static_cast<T*>(a.dz) + t * a.dz_ld;
    float w = 0.0f;
    if (mass && !bad) {
      w = a.temperature;
      if (a.mean) w /= static_cast<float>(a.st->count);
      if (a.row_grad != nullptr) w *= a.row_grad[t];
    }
    const float ws = w / s;
    const T* z0 = z + s0 - mis;
    T* out0 = out + s0 - mis;
    const bool vec = (reinterpret_cast<uintptr_t>(out0) % 16) == 0;
    const bool live = mass && !bad;
    for (int j = threadIdx.x; j < nvec; j += kDistillThreads) {
      const bool whole = (j > 0 || mis == 0) && (j + 1) * VEC <= s1 - s0 + mis;
      uint4 raw = make_uint4(0, 0, 0, 0), res = make_uint4(0, 0, 0, 0);
      const T* o = reinterpret_cast<const T*>(&raw);
      T* d = reinterpret_cast<T*>(&res);
      if (live) {
        if (a.cached) {
          raw = reinterpret_cast<const uint4*>(cache)[j];
        } else if (whole) {
          raw = reinterpret_cast<const uint4*>(z0)[j];
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int c = j * VEC + i;
            if (c >= mis && c < s1 - s0 + mis) reinterpret_cast<T*>(&raw)[i] = z0[c];
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) from_f32(ws * ex2((to_f32(o[i]) - m) * scale2), d[i]);
      }
      if (whole && vec) {
        __stcs(reinterpret_cast<uint4*>(out0) + j, res);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int c = j * VEC + i;
          if (c >= mis && c < s1 - s0 + mis) out0[c] = d[i];
        }
      }
    }
    // The entries' places again, with q taken off before the one rounding.
    __syncthreads();
    if (live) {
      for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
        const int c = si[k];
        if (c < s0 || c >= s1) continue;
        float goal = 0.0f;
        bool first = true;
        for (int j = 0; j < a.top; ++j) {
          if (si[j] != c) continue;
          first = first && j >= k;
          goal += sq[j];
        }
        if (first) from_f32(w * (ex2((sz[k] - m) * scale2) / s - goal), out[c]);
      }
    }
  }
  if (cs > 1 && mass && !bad) cluster_sync();  // no CTA leaves while another reads its share

  if (a.loss == nullptr || rank != 0) return;
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(&a.st->done, 1u) == static_cast<unsigned int>(a.T) - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
  for (long long r = threadIdx.x; r < a.T; r += kDistillThreads) sum += static_cast<double>(__ldcg(a.loss_rows + r));
  sum = block_sum(sum, dbuf);
  if (threadIdx.x == 0) {
    if (a.mean) sum /= static_cast<double>(a.st->count > 0 ? a.st->count : 1);
    *a.loss = static_cast<float>(sum);
  }
}

template <int DT, bool GRAD>
int launch_distill(const DistillArgs& a, int cs, size_t smem, cudaStream_t s) {
  auto kern = distill_kernel<DT, GRAD>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return set_error(PO_ERR_CUDA, "device ordinal out of range");
  if (!configured[dev]) {
    const int r = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 120 << 10),
                             "cudaFuncSetAttribute");
    if (r) return r;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.T * cs), 1, 1);
  cfg.blockDim = dim3(kDistillThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a), "distill launch");
}

template <int DT>
__global__ void __launch_bounds__(256) scale_kernel(void* x, long long n, const float* factor) {
  using T = typename ElemOf<DT>::T;
  const float f = *factor;
  if (f == 1.0f) return;
  T* p = static_cast<T*>(x);
  constexpr int VEC = 16 / sizeof(T);
  const long long first = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long nv = reinterpret_cast<uintptr_t>(x) % 16 == 0 ? n / VEC : 0;
  for (long long i = first; i < nv; i += step) {
    uint4 raw = reinterpret_cast<uint4*>(x)[i];
    T* o = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int k = 0; k < VEC; ++k) from_f32(to_f32(o[k]) * f, o[k]);
    reinterpret_cast<uint4*>(x)[i] = raw;
  }
  for (long long i = nv * VEC + first; i < n; i += step) from_f32(to_f32(p[i]) * f, p[i]);
}

}  // namespace
}  // namespace po

using namespace po;

extern "C" size_t po_distill_logits_workspace_bytes(long long tokens) { return tokens > 0 ? sizeof(DistillState) : 0; }

extern "C" int po_distill_logits(const void* logits, long long ld, int dtype, long long tokens, long long vocab,
                                 const long long* index, long long index_ld, const void* teacher, long long teacher_ld,
                                 int teacher_dtype, long long top, float temperature, int mean, const float* row_grad,
                                 float* loss_rows, float* loss, void* dlogits, long long dl_ld, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (dtype != PO_F32 && dtype != PO_BF16 && dtype != PO_F16)
    return set_error(PO_ERR_ARG, "distill_logits: dtype must be fp32, bf16 or fp16");
  if (teacher_dtype != PO_F32 && teacher_dtype != PO_BF16 && teacher_dtype != PO_F16)
    return set_error(PO_ERR_ARG, "distill_logits: teacher dtype must be fp32, bf16 or fp16");
  if (tokens < 0 || tokens > (1 << 26) || vocab <= 0 || vocab > (1 << 28))
    return set_error(PO_ERR_ARG, "distill_logits: bad size");
  if (top < 1 || top > kMaxTop) return set_error(PO_ERR_ARG, "distill_logits: top must be 1 to 1024");
  if (!(temperature > 0.0f) || !std::isfinite(temperature))
    return set_error(PO_ERR_ARG, "distill_logits: temperature must be positive");
  if (row_grad != nullptr && (mean || dlogits == nullptr))
    return set_error(PO_ERR_ARG, "distill_logits: row_grad goes with gradients of the sum");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tokens == 0) return loss == nullptr ? PO_OK : check_cuda(cudaMemsetAsync(loss, 0, 4, s), "distill_logits");
  if (tokens > 1 && (ld < vocab || index_ld < top || teacher_ld < top || (dlogits != nullptr && dl_ld < vocab)))
    return set_error(PO_ERR_ARG, "distill_logits: a pitch is smaller than its row");
  if (logits == nullptr || index == nullptr || teacher == nullptr || loss_rows == nullptr)
    return set_error(PO_ERR_ARG, "distill_logits: null operand");
  DistillArgs a{};
  a.z = logits, a.ld = ld, a.dz = dlogits, a.dz_ld = dl_ld, a.T = tokens, a.V = static_cast<int>(vocab);
  a.index = index, a.index_ld = index_ld, a.teacher = teacher, a.teacher_ld = teacher_ld;
  a.teacher_dtype = teacher_dtype, a.top = static_cast<int>(top), a.temperature = temperature, a.mean = mean;
  a.row_grad = row_grad, a.loss_rows = loss_rows, a.loss = loss;
  if (loss != nullptr || mean) {
    if (workspace == nullptr || workspace_bytes < sizeof(DistillState))
      return set_error(PO_ERR_WORKSPACE, "distill_logits: workspace too small");
    a.st = static_cast<DistillState*>(workspace);
    if (int r = check_cuda(cudaMemsetAsync(a.st, 0, sizeof(DistillState), s), "distill_logits")) return r;
  }
  if (mean) {
    const int blocks = cdiv(tokens, 8) < 2 * sm_count() ? cdiv(tokens, 8) : 2 * sm_count();
    count_rows_kernel<<<blocks, 256, 0, s>>>(a);
    if (int r = check_cuda(cudaGetLastError(), "distill_logits count")) return r;
  }
  // CTAs a row: segments of at most 32 KB (several CTAs on an SM), and all 8
  // when there are too few rows to fill the SMs otherwise.
  const int es = dtype_size(dtype);
  int cs = 1;
  while (cs < 8 && (vocab * es > cs * (32LL << 10) || (tokens * cs < 2 * sm_count() && vocab > cs * 2048LL))) cs *= 2;
  const int vec = 16 / es;
  a.seg = static_cast<int>(round_up((vocab + cs - 1) / cs, vec));
  const size_t entries = (static_cast<size_t>(top) * 12 + 15) / 16 * 16;
  const size_t seg_bytes = static_cast<size_t>(a.seg + 2 * vec) * es;
  a.cached = dlogits != nullptr && seg_bytes <= (96u << 10);
  const size_t smem = entries + (a.cached ? seg_bytes : 0);
  const bool g = dlogits != nullptr;
  if (dtype == PO_F32) return g ? launch_distill<PO_F32, true>(a, cs, smem, s) : launch_distill<PO_F32, false>(a, cs, smem, s);
  if (dtype == PO_BF16)
    return g ? launch_distill<PO_BF16, true>(a, cs, smem, s) : launch_distill<PO_BF16, false>(a, cs, smem, s);
  return g ? launch_distill<PO_F16, true>(a, cs, smem, s) : launch_distill<PO_F16, false>(a, cs, smem, s);
}

extern "C" int po_scale_inplace(void* x, int dtype, long long n, const float* factor, void* stream) {
  if (dtype != PO_F32 && dtype != PO_BF16 && dtype != PO_F16)
    return set_error(PO_ERR_ARG, "scale_inplace: dtype must be fp32, bf16 or fp16");
  if (n < 0) return set_error(PO_ERR_ARG, "scale_inplace: negative size");
  if (n == 0) return PO_OK;
  if (x == nullptr || factor == nullptr) return set_error(PO_ERR_ARG, "scale_inplace: null operand");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long want = (n + 2047) / 2048;
  const int blocks = static_cast<int>(want < 8LL * sm_count() ? want : 8LL * sm_count());
  if (dtype == PO_F32) scale_kernel<PO_F32><<<blocks, 256, 0, s>>>(x, n, factor);
  else if (dtype == PO_BF16) scale_kernel<PO_BF16><<<blocks, 256, 0, s>>>(x, n, factor);
  else scale_kernel<PO_F16><<<blocks, 256, 0, s>>>(x, n, factor);
  return check_cuda(cudaGetLastError(), "scale_inplace");
}
