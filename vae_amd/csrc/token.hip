// Log probabilities of given tokens, entropy and top alternatives of rows of logits [N, V], their gradient, and the
// categorical NLL's loss gradient.  Formulas and the conventions for masks: token_row.hpp.
//   log p_t,   H = ln2 (log2 s - sum d 2^d / s) with d = (x - m) log2(e),   top k by (value, lower index first)
//   dx_j = sum_i g_i ([j = id_i] - p_j) - g_H p_j (ln p_j + H)       (i: the token and the alternatives)
// A row whose token is negative is padding: none of its logits is read.
#include "token_row.hpp"
#include "../../include/vae_amd.h"

namespace vae {

constexpr int kMaxGrid = 1 << 20;  // blocks of a launch; rows beyond are grid-strided

template <typename T>
__global__ __launch_bounds__(kBlock) void token_fwd_kernel(
    const T* __restrict__ logits, int64_t row_stride, const void* __restrict__ tokens, int token_bytes,
    float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_logp,
    int64_t* __restrict__ top_ids, int top_k, int64_t N, int V) {
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* x = logits + row * row_stride;
    const int64_t tok = tokens ? load_id(tokens, token_bytes, row) : 0;
    if (tok < 0) {
      if (threadIdx.x == 0) {
        if (logp) logp[row] = 0.f;
        if (entropy) entropy[row] = 0.f;
        if (stats) stats[2 * row] = stats[2 * row + 1] = 0.f;
      }
      for (int i = threadIdx.x; i < top_k; i += kBlock) {
        top_logp[row * top_k + i] = -INFINITY;
        top_ids[row * top_k + i] = -1;
      }
      continue;
    }
    float m = kLowest;
    for (int j = threadIdx.x; j < V; j += kBlock) m = fmaxf(m, to_f32(x[j]));
    m = row_max(m, kBlock);
    float s = 0.f, t = 0.f;
    for (int j = threadIdx.x; j < V; j += kBlock) {
      const float d = (to_f32(x[j]) - m) * kLog2e;
      const float e = __builtin_amdgcn_exp2f(d);
      s += e;
      t += fmaxf(d, -300.f) * e;
    }
    s = row_sum(s, kBlock);
    t = row_sum(t, kBlock);
    uint64_t last = ~0ull;
    for (int i = 0; i < top_k; ++i) {
      uint64_t best = 0;
      for (int j = threadIdx.x; j < V; j += kBlock) {
        const uint64_t k = order_key(to_f32(x[j]), j);
        if (k < last && k > best) best = k;
      }
      last = block_max_u64(best);
      if (threadIdx.x == 0) {
        const bool some = (last >> 32) != 0;
        top_logp[row * top_k + i] = some ? row_log_prob(order_value(last >> 32), m, s, 1.0f) : nan_f();
        top_ids[row * top_k + i] = some ? (int64_t)(uint32_t)~(uint32_t)last : -1;
      }
    }
    if (threadIdx.x == 0) {
      if (logp) logp[row] = tok < V ? row_log_prob(to_f32(x[tok]), m, s, 1.0f) : nan_f();
      if (entropy) entropy[row] = s == 0.f ? 0.f : kLn2 * (log2f(s) - t / s);
      if (stats) {
        stats[2 * row] = m;
        stats[2 * row + 1] = s;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void token_bwd_kernel(
    const T* __restrict__ logits, int64_t row_stride, const void* __restrict__ tokens, int token_bytes,
    const float* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ glogp,
    int64_t rows_per_g, float g_scale, const float* __restrict__ gentropy, const float* __restrict__ gtop,
    const int64_t* __restrict__ top_ids, int top_k, T* __restrict__ glogits, int64_t N, int V) {
  for (int64_t row = blockIdx.x; row < N; row += gridDim.x) {
    const T* x = logits + row * row_stride;
    T* gx = glogits + row * (int64_t)V;
    const int64_t tok = tokens ? load_id(tokens, token_bytes, row) : 0;
    const float m = stats[2 * row], s = stats[2 * row + 1];
    if (tok < 0 || s == 0.f) {
      for (int j = threadIdx.x; j < V; j += kBlock) gx[j] = from_f32<T>(0.f);
      continue;
    }
    float gt = tokens ? (glogp ? glogp[row / rows_per_g] * g_scale : g_scale) : 0.f;
    if (tok >= V) gt *= nan_f();
    const float gh = gentropy ? gentropy[row] : 0.f, h = gentropy ? entropy[row] : 0.f;
    float a = gt;
    for (int i = 0; i < top_k; ++i) a += gtop[row * top_k + i];
    const float inv = 1.0f / s, ls = log2f(s);
    for (int j = threadIdx.x; j < V; j += kBlock) {
      const float d = (to_f32(x[j]) - m) * kLog2e;
      const float p = __builtin_amdgcn_exp2f(d) * inv;
      float g = -p * (a + gh * (h + kLn2 * (fmaxf(d, -300.f) - ls)));
      if (j == tok) g += gt;
      for (int i = 0; i < top_k; ++i)
        if (top_ids[row * top_k + i] == j) g += gtop[row * top_k + i];
      gx[j] = from_f32<T>(g);
    }
  }
}

// out[b] = scale * sum of T consecutive row values, in a fixed order, summed in double
template <typename O>
__global__ __launch_bounds__(kBlock) void row_sums_kernel(const float* __restrict__ rows, float scale,
                                                          O* __restrict__ out, int64_t B, int64_t T) {
  __shared__ double part[kBlock / 64];
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    double v = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += kBlock) v += (double)rows[b * T + t];
    v = wave_sum_d(v);
    lds_barrier();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    lds_barrier();
    if (threadIdx.x == 0) {
      double r = 0.0;
      for (int w = 0; w < kBlock / 64; ++w) r += part[w];
      out[b] = from_f32<O>((float)(r * (double)scale));
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void grad_scale_kernel(T* __restrict__ buf, const float* __restrict__ factor,
                                                            int64_t items) {
  const float c = factor[0];
  if (c == 1.0f) return;
  for (int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x; j < items; j += (int64_t)gridDim.x * kBlock) {
    float v[V];
    load_vec<T, V, false>(buf + j * V, v);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= c;
    store_vec<T, V>(buf + j * V, v);
  }
}

static bool bad_shape(int64_t N, int64_t V, int64_t row_stride, int dtype) {
  return N < 0 || V < 1 || V > VAE_MAX_ROW || (N > 1 && row_stride < V) ||
         (dtype != VAE_F32 && dtype != VAE_BF16 && dtype != VAE_F16);
}
static int row_grid(int64_t rows) { return (int)(rows < kMaxGrid ? rows : kMaxGrid); }

template <typename T>
static int token_fwd_type(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp,
                          float* entropy, float* stats, float* top_logp, int64_t* top_ids, int64_t top_k, int64_t N,
                          int64_t V, hipStream_t st) {
  hipLaunchKernelGGL((token_fwd_kernel<T>), dim3(row_grid(N)), dim3(kBlock), 0, st, (const T*)logits, row_stride, tokens,
                     token_bytes, logp, entropy, stats, top_logp, top_ids, (int)top_k, N, (int)V);
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
}

template <typename T>
static int token_bwd_type(const void* logits, int64_t row_stride, const void* tokens, int token_bytes,
                          const float* stats, const float* entropy, const float* glogp, int64_t rows_per_g,
                          float g_scale, const float* gentropy, const float* gtop, const int64_t* top_ids,
                          int64_t top_k, void* glogits, int64_t N, int64_t V, hipStream_t st) {
  hipLaunchKernelGGL((token_bwd_kernel<T>), dim3(row_grid(N)), dim3(kBlock), 0, st, (const T*)logits, row_stride, tokens,
                     token_bytes, stats, entropy, glogp, rows_per_g, g_scale, gentropy, gtop, top_ids, (int)top_k,
                     (T*)glogits, N, (int)V);
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
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

int vae_token_logp_fwd(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp,
                       float* entropy, float* stats, float* top_logp, int64_t* top_ids, int64_t top_k, int64_t N,
                       int64_t V, int dtype, vae_stream_t stream) {
  if (bad_shape(N, V, row_stride, dtype) || top_k < 0 || top_k > VAE_MAX_TOP || top_k > V) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || (tokens && token_bytes != 4 && token_bytes != 8)) return VAE_ERR_ARG;
  if ((logp && !tokens) || (top_k > 0 && (!top_logp || !top_ids))) return VAE_ERR_ARG;
  VAE_BY_TYPE(dtype, return token_fwd_type<T>(logits, row_stride, tokens, token_bytes, logp, entropy, stats, top_logp,
                                              top_ids, top_k, N, V, (hipStream_t)stream));
  return VAE_ERR_ARG;
}

int vae_token_logp_bwd(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, const float* stats,
                       const float* entropy, const float* glogp, int64_t rows_per_g, float g_scale,
                       const float* gentropy, const float* gtop, const int64_t* top_ids, int64_t top_k, void* glogits,
                       int64_t N, int64_t V, int dtype, vae_stream_t stream) {
  if (bad_shape(N, V, row_stride, dtype) || top_k < 0 || top_k > VAE_MAX_TOP || rows_per_g < 1) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !stats || !glogits || (tokens && token_bytes != 4 && token_bytes != 8)) return VAE_ERR_ARG;
  if ((gentropy && !entropy) || (top_k > 0 && (!gtop || !top_ids)) || (glogp && !tokens)) return VAE_ERR_ARG;
  VAE_BY_TYPE(dtype, return token_bwd_type<T>(logits, row_stride, tokens, token_bytes, stats, entropy, glogp,
                                              rows_per_g, g_scale, gentropy, gtop, top_ids, top_k, glogits, N, V,
                                              (hipStream_t)stream));
  return VAE_ERR_ARG;
}

int vae_token_nll_fused(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp,
                        float* stats, void* glogits, float grad_scale, int64_t N, int64_t V, int dtype,
                        vae_stream_t stream) {
  if (N > 0 && (!tokens || !logp || !stats || !glogits)) return VAE_ERR_ARG;
  const int rc = vae_token_logp_fwd(logits, row_stride, tokens, token_bytes, logp, nullptr, stats, nullptr, nullptr, 0,
                                    N, V, dtype, stream);
  if (rc != VAE_OK) return rc;
  return vae_token_logp_bwd(logits, row_stride, tokens, token_bytes, stats, nullptr, nullptr, 1, -grad_scale, nullptr,
                            nullptr, nullptr, 0, glogits, N, V, dtype, stream);
}

int vae_row_sums(const float* rows, float scale, void* out, int64_t B, int64_t T_, int dtype, vae_stream_t stream) {
  if (B < 0 || T_ < 0) return VAE_ERR_ARG;
  if (B == 0) return VAE_OK;
  if (!out || (T_ > 0 && !rows)) return VAE_ERR_ARG;
  VAE_BY_TYPE(dtype, hipLaunchKernelGGL((row_sums_kernel<T>), dim3(row_grid(B)), dim3(kBlock), 0, (hipStream_t)stream,
                                        rows, scale, (T*)out, B, T_);
              return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH);
  return VAE_ERR_ARG;
}

int vae_grad_scale(void* buf, const float* factor, int64_t n, int dtype, vae_stream_t stream) {
  if (n < 0) return VAE_ERR_ARG;
  if (n == 0) return VAE_OK;
  if (!buf || !factor) return VAE_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  VAE_BY_TYPE(dtype, constexpr int VN = VecOf<T>::n; const bool vec = n % VN == 0 && aligned16(buf);
              const int64_t items = vec ? n / VN : n; const int64_t blocks = (items + kBlock - 1) / kBlock;
              const int grid = (int)(blocks < 4096 ? blocks : 4096);
              if (vec) hipLaunchKernelGGL((grad_scale_kernel<T, VN>), dim3(grid), dim3(kBlock), 0, st, (T*)buf, factor, items);
              else hipLaunchKernelGGL((grad_scale_kernel<T, 1>), dim3(grid), dim3(kBlock), 0, st, (T*)buf, factor, items);
              return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH);
  return VAE_ERR_ARG;
}

}  // extern "C"
