// Distillation from a teacher's top logits: per row, the teacher's K largest logits y_k with their ids and the
// student's row x[V], both at temperature tau:
//   q = softmax(y / tau) over the entries that are there (id >= 0, logit > -inf),  p = softmax(x / tau) over V,
//   KL = sum_k q_k (ln q_k - ln p_id_k),      dx_j = (g / tau) (p_j - sum_{k: id_k = j} q_k).
// The same id may come twice; a row with no entry left has KL 0 and gradient 0.  Row statistics: token_row.hpp.
#include "token_row.hpp"
#include "../../include/vae_amd.h"

namespace vae {

constexpr int kMaxGrid = 1 << 20;  // blocks of a launch; rows beyond are grid-strided

__device__ __forceinline__ float load_any(const void* __restrict__ p, int dtype, int64_t i) {
  if (dtype == VAE_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == VAE_BF16) return to_f32(reinterpret_cast<const bf16_t*>(p)[i]);
  return to_f32(reinterpret_cast<const f16_t*>(p)[i]);
}

// The teacher's row in LDS: ids (-1: absent), q and ln q.  state: 0 fine, 1 nothing there, 2 an id beyond the vocabulary.
struct TeacherRow {
  int id[VAE_MAX_TEACHER];
  float q[VAE_MAX_TEACHER], logq[VAE_MAX_TEACHER];
};
__device__ __forceinline__ int load_teacher(TeacherRow& tr, const void* __restrict__ t_logits, int64_t t_stride,
                                            int t_dtype, const void* __restrict__ t_ids, int64_t id_stride, int id_bytes,
                                            int K, int64_t row, int V, float inv_tau, float scale2) {
  const int k = threadIdx.x;
  float y = -INFINITY;
  int id = -1;
  bool bad = false;
  lds_barrier();  // the row before this one has been read
  if (k < K) {
    const int64_t i = load_id(t_ids, id_bytes, row * id_stride + k);
    bad = i >= V;
    if (i >= 0 && !bad) {
      y = load_any(t_logits, t_dtype, row * t_stride + k);
      id = (int)i;
    }
  }
  const float m = row_max(fmaxf(y, kLowest), kBlock);
  const float d = (y - m) * scale2;
  const float e = id >= 0 ? __builtin_amdgcn_exp2f(d) : 0.f;
  const float s = row_sum(e, kBlock);
  const float any_bad = row_sum(bad ? 1.f : 0.f, kBlock);
  if (k < K) {
    tr.q[k] = e / s;
    tr.logq[k] = row_log_prob(y, m, s, inv_tau);
    tr.id[k] = (e == 0.f) ? -1 : id;   // e NaN keeps its id: the row comes out NaN
  }
  lds_barrier();
  return any_bad > 0.f ? 2 : (s == 0.f ? 1 : 0);
}

template <typename T>
__global__ __launch_bounds__(kBlock) void distill_fwd_kernel(
    const T* __restrict__ logits, int64_t row_stride, const void* __restrict__ t_logits, int64_t t_stride, int t_dtype,
    const void* __restrict__ t_ids, int64_t id_stride, int id_bytes, int K, float inv_tau, float scale2, float* __restrict__ kl,
    float* __restrict__ stats, int64_t N, int V) {
  __shared__ TeacherRow tr;
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* x = logits + row * row_stride;
    const int state = load_teacher(tr, t_logits, t_stride, t_dtype, t_ids, id_stride, id_bytes, K, row, V, inv_tau, scale2);
    if (state) {
      if (threadIdx.x == 0) {
        kl[row] = state == 1 ? 0.f : nan_f();
        if (stats) stats[2 * row] = stats[2 * row + 1] = 0.f;
      }
      continue;
    }
    float m = kLowest;
    for (int j = threadIdx.x; j < V; j += kBlock) m = fmaxf(m, to_f32(x[j]));
    m = row_max(m, kBlock);
    float s = 0.f;
    for (int j = threadIdx.x; j < V; j += kBlock) s += __builtin_amdgcn_exp2f((to_f32(x[j]) - m) * scale2);
    s = row_sum(s, kBlock);
    float v = 0.f;
    if (threadIdx.x < K && tr.id[threadIdx.x] >= 0)
      v = tr.q[threadIdx.x] * (tr.logq[threadIdx.x] - row_log_prob(to_f32(x[tr.id[threadIdx.x]]), m, s, inv_tau));
    v = row_sum(v, kBlock);
    if (threadIdx.x == 0) {
      kl[row] = v;
      if (stats) {
        stats[2 * row] = m;
        stats[2 * row + 1] = s;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void distill_bwd_kernel(
    const T* __restrict__ logits, int64_t row_stride, const void* __restrict__ t_logits, int64_t t_stride, int t_dtype,
    const void* __restrict__ t_ids, int64_t id_stride, int id_bytes, int K, float inv_tau, float scale2,
    const float* __restrict__ stats, const float* __restrict__ gkl, const float* __restrict__ gmean, float mean_scale,
    T* __restrict__ glogits, int64_t N, int V) {
  __shared__ TeacherRow tr;
  const float g0 = gmean ? gmean[0] * mean_scale : (gkl ? 0.f : mean_scale);
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* x = logits + row * row_stride;
    T* gx = glogits + row * (int64_t)V;
    const int state = load_teacher(tr, t_logits, t_stride, t_dtype, t_ids, id_stride, id_bytes, K, row, V, inv_tau, scale2);
    const float m = stats[2 * row], s = stats[2 * row + 1];
    float c = ((gkl ? gkl[row] : 0.f) + g0) * inv_tau;
    if (state == 2) c = nan_f();
    if (state == 1 || (state == 0 && s == 0.f)) {
      for (int j = threadIdx.x; j < V; j += kBlock) gx[j] = from_f32<T>(0.f);
      continue;
    }
    const float inv = 1.0f / s;
    for (int j = threadIdx.x; j < V; j += kBlock) {
      float g = __builtin_amdgcn_exp2f((to_f32(x[j]) - m) * scale2) * inv;
      for (int k = 0; k < K; ++k)
        if (tr.id[k] == j) g -= tr.q[k];
      gx[j] = from_f32<T>(state == 2 ? c : c * g);
    }
  }
}

static int row_grid(int64_t rows) { return (int)(rows < kMaxGrid ? rows : kMaxGrid); }
static bool bad_args(int64_t N, int64_t V, int64_t row_stride, int dtype, int64_t t_stride, int t_dtype,
                     int64_t id_stride, int id_bytes, int64_t K, float temperature) {
  auto type_ok = [](int d) { return d == VAE_F32 || d == VAE_BF16 || d == VAE_F16; };
  return N < 0 || V < 1 || V > VAE_MAX_ROW || (N > 1 && row_stride < V) || !type_ok(dtype) || !type_ok(t_dtype) ||
         K < 1 || K > VAE_MAX_TEACHER || (N > 1 && (t_stride < K || id_stride < K)) ||
         (id_bytes != 4 && id_bytes != 8) || !(temperature > 0.f) || !(temperature < INFINITY);
}

}  // namespace vae

using namespace vae;

#define VAE_BY_TYPE(dtype_, ...)                                        \
  switch (dtype_) {                                                     \
    case VAE_F32: { using T = float; __VA_ARGS__; } break;              \
    case VAE_BF16: { using T = bf16_t; __VA_ARGS__; } break;            \
    case VAE_F16: { using T = f16_t; __VA_ARGS__; } break;              \
  }

extern "C" {

int vae_distill_bwd(const void* logits, int64_t row_stride, const void* t_logits, int64_t t_stride, int t_dtype,
                    const void* t_ids, int64_t id_stride, int id_bytes, int64_t K, float temperature,
                    const float* stats, const float* gkl, const float* gmean, float mean_scale, void* glogits,
                    int64_t N, int64_t V, int dtype, vae_stream_t stream) {
  if (bad_args(N, V, row_stride, dtype, t_stride, t_dtype, id_stride, id_bytes, K, temperature)) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !t_logits || !t_ids || !stats || !glogits) return VAE_ERR_ARG;
  const float scale2 = (float)(1.4426950408889634 / (double)temperature);
  const float inv_tau = (float)(1.0 / (double)temperature);
  VAE_BY_TYPE(dtype, hipLaunchKernelGGL((distill_bwd_kernel<T>), dim3(row_grid(N)), dim3(kBlock), 0, (hipStream_t)stream,
                                        (const T*)logits, row_stride, t_logits, t_stride, t_dtype, t_ids, id_stride,
                                        id_bytes, (int)K, inv_tau, scale2, stats, gkl, gmean, mean_scale, (T*)glogits,
                                        N, (int)V);
              return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH);
  return VAE_ERR_ARG;
}

int vae_distill_fwd(const void* logits, int64_t row_stride, const void* t_logits, int64_t t_stride, int t_dtype,
                    const void* t_ids, int64_t id_stride, int id_bytes, int64_t K, float temperature, float* kl,
                    float* stats, void* glogits, float grad_scale, int64_t N, int64_t V, int dtype,
                    vae_stream_t stream) {
  if (bad_args(N, V, row_stride, dtype, t_stride, t_dtype, id_stride, id_bytes, K, temperature)) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !t_logits || !t_ids || !kl || (glogits && !stats)) return VAE_ERR_ARG;
  const float scale2 = (float)(1.4426950408889634 / (double)temperature);
  const float inv_tau = (float)(1.0 / (double)temperature);
  VAE_BY_TYPE(dtype, hipLaunchKernelGGL((distill_fwd_kernel<T>), dim3(row_grid(N)), dim3(kBlock), 0, (hipStream_t)stream,
                                        (const T*)logits, row_stride, t_logits, t_stride, t_dtype, t_ids, id_stride,
                                        id_bytes, (int)K, inv_tau, scale2, kl, stats, N, (int)V));
  if (hipGetLastError() != hipSuccess) return VAE_ERR_LAUNCH;
  if (!glogits) return VAE_OK;
  return vae_distill_bwd(logits, row_stride, t_logits, t_stride, t_dtype, t_ids, id_stride, id_bytes, K, temperature,
                         stats, nullptr, nullptr, grad_scale, glogits, N, V, dtype, stream);
}

}  // extern "C"
