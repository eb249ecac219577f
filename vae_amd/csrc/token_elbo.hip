// What closes a categorical likelihood: the samples' sums of their tokens' log probs, the ELBO combine with its six batch
// means, and the backward of both; sums of row values; a stored gradient times a device scalar.  All of it is [B] or
// [rows] work of a few microseconds: one launch each.
#include "token_row.hpp"

namespace vae {

// The six means leave the first launch as block partials in the caller's `means` buffer and a second one adds them, in
// block order and in double; a single block writes them itself.  No counters, so calls and captured graphs share nothing
// (the saw-a-NaN word of the workspace is a bit that several may set).
constexpr int kElboBlocks = 256;
constexpr int kOneBlock = 1024;
static_assert(VAE_TOKEN_MEANS_FLOATS == 6 + 6 * kElboBlocks, "the header says how long `means` is");

__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == VAE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == VAE_BF16) reinterpret_cast<bf16_t*>(p)[i] = from_f32<bf16_t>(v);
  else reinterpret_cast<f16_t*>(p)[i] = from_f32<f16_t>(v);
}
// where the caller wants the means, in its own type; each may be NULL
struct MeansTo {
  void *loss, *others;
  int dtype;
};
// thread k < 6: total k -> mean k
__device__ __forceinline__ void write_mean(int k, double total, float inv_count, float* means, const MeansTo& to,
                                           float* ws) {
  const float v = (float)(total * (double)inv_count);
  means[k] = v;
  if (k == 0 && to.loss) store_any(to.loss, to.dtype, 0, v);
  if (k > 0 && to.others) store_any(to.others, to.dtype, k - 1, v);
  if (ws) note_nan(ws, v, kNanElbo6, k);
}

// `len` values p[first], p[first + step], ... in double; eight loads on their way at a time
__device__ __forceinline__ double strided_sum(const float* __restrict__ p, int64_t first, int64_t step, int64_t len) {
  double v = 0.0;
  int64_t t = first;
  for (; t + 7 * step < len; t += 8 * step) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[t + i * step];
#pragma unroll
    for (int i = 0; i < 8; ++i) v += (double)x[i];
  }
  for (; t < len; t += step) v += (double)p[t];
  return v;
}

// the ELBO's terms [B] beside the nll, in the type that they come in; each may be NULL
struct Terms {
  const void *kld, *add, *mi;
  int dtype;
};

// G lanes a sample (a power of two, up to a wave); samples in order, so a result does not depend on timing
template <typename T, int BT>
__global__ __launch_bounds__(BT) void token_elbo_fwd_kernel(
    const float* __restrict__ logp, int64_t len, Terms terms, float kl_beta, float inv_count, T* __restrict__ nll,
    T* __restrict__ loss, T* __restrict__ elbo, float* __restrict__ means, MeansTo to, float* __restrict__ ws, int64_t B,
    int G) {
  __shared__ float part[BT / 64][6];
  const int rpb = BT / G, sub = threadIdx.x % G, rloc = threadIdx.x / G;
  float acc[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t b0 = (int64_t)blockIdx.x * rpb; b0 < B; b0 += (int64_t)gridDim.x * rpb) {
    const int64_t b = b0 + rloc;
    double v = b < B ? strided_sum(logp + b * len, sub, G, len) : 0.0;
    for (int o = G >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if (sub != 0 || b >= B) continue;
    const float n = (float)(0.0 - v);   // loss and elbo from the unrounded sum: every output is rounded once
    if (nll) nll[b] = from_f32<T>(n);
    if (!loss) continue;
    const float k = terms.kld ? load_any(terms.kld, terms.dtype, b) : 0.f;
    const float ad = terms.add ? load_any(terms.add, terms.dtype, b) : 0.f;
    const float m = terms.mi ? load_any(terms.mi, terms.dtype, b) : 0.f;
    const float e = n + k, l = (n + ad + kl_beta * k) - m;
    loss[b] = from_f32<T>(l);
    elbo[b] = from_f32<T>(e);
    acc[0] += l; acc[1] += e; acc[2] += n; acc[3] += k; acc[4] += ad; acc[5] += m;
  }
  if (!loss) return;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const float s = wave_total(acc[k]);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][k] = s;
  }
  lds_barrier();
  if (threadIdx.x < 6) {
    const int k = threadIdx.x;
    float s = 0.f;
    for (int w = 0; w < BT / 64; ++w) s += part[w][k];
    if (gridDim.x == 1) write_mean(k, s, inv_count, means, to, ws);
    else means[6 + 6 * blockIdx.x + k] = s;
  }
}
__global__ __launch_bounds__(64) void token_elbo_means_kernel(float* __restrict__ means, int blocks, float inv_count,
                                                              MeansTo to, float* __restrict__ ws) {
  for (int k = 0; k < 6; ++k) {
    double v = 0.0;
    for (int b = threadIdx.x; b < blocks; b += 64) v += (double)means[6 + 6 * b + k];
    v = wave_sum_d(v);
    if ((int)threadIdx.x == k) write_mean(k, v, inv_count, means, to, ws);
  }
}

struct Scalars6 {
  const void* p[6];
};
// where the terms' gradients go, in the terms' type; each may be NULL
struct GradTerms {
  void *kld, *add, *mi;
  int dtype;
};
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void token_elbo_bwd_kernel(
    const T* __restrict__ gnll, const T* __restrict__ gloss, const T* __restrict__ gelbo, Scalars6 gmeans,
    int gmeans_dtype, float kl_beta, float inv_count, float* __restrict__ grow, T* __restrict__ grad, int64_t items,
    GradTerms gterms, int64_t B) {
  float gm[6];
#pragma unroll
  for (int k = 0; k < 6; ++k) gm[k] = gmeans.p[k] ? load_any(gmeans.p[k], gmeans_dtype, 0) : 0.f;
  const float c = gm[0] + gm[1] + gm[2];
  for (int64_t b = (int64_t)blockIdx.x * kBlock + threadIdx.x; b < B; b += (int64_t)gridDim.x * kBlock) {
    const float gl = (gloss ? to_f32(gloss[b]) : 0.f) + gm[0] * inv_count;
    const float ge = (gelbo ? to_f32(gelbo[b]) : 0.f) + gm[1] * inv_count;
    if (grow) grow[b] = gl + ge + gm[2] * inv_count + (gnll ? to_f32(gnll[b]) : 0.f);
    if (gterms.kld) store_any(gterms.kld, gterms.dtype, b, kl_beta * gl + ge + gm[3] * inv_count);
    if (gterms.add) store_any(gterms.add, gterms.dtype, b, gl + gm[4] * inv_count);
    if (gterms.mi) store_any(gterms.mi, gterms.dtype, b, gm[5] * inv_count - gl);
  }
  if (!grad || c == 1.0f) return;
  for (int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x; j < items; j += (int64_t)gridDim.x * kBlock) {
    float v[V];
    load_vec<T, V, false>(grad + j * V, v);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= c;
    store_vec<T, V>(grad + j * V, v);
  }
}

// out[b] = scale * sum of `len` consecutive row values, in a fixed order, summed in double: a workgroup a sum.  One sum
// over everything (a mean over all rows) is bound by its loads' latency: 1024 threads, eight loads each on their way
// (65536 values: 60 us with 256 threads and a load at a time).
template <typename O, int BT>
__global__ __launch_bounds__(BT) void row_sums_kernel(const float* __restrict__ rows, float scale,
                                                          O* __restrict__ out, int64_t B, int64_t len) {
  __shared__ double part[BT / 64];
  for (int64_t b = blockIdx.x; b < B; b += gridDim.x) {
    const double v = wave_sum_d(strided_sum(rows + b * len, threadIdx.x, BT, len));
    lds_barrier();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    lds_barrier();
    if (threadIdx.x == 0) {
      double r = 0.0;
      for (int w = 0; w < BT / 64; ++w) r += part[w];
      out[b] = from_f32<O>((float)(r * (double)scale));
    }
  }
}

static int launched() { return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH; }
static bool type_ok(int d) { return d == VAE_F32 || d == VAE_BF16 || d == VAE_F16; }

template <typename T, int V>
static void elbo_bwd_launch(const void* gnll, const void* gloss, const void* gelbo, const Scalars6& gm, int gmeans_dtype,
                            float kl_beta, float inv_count, float* grow, void* grad, int64_t items,
                            const GradTerms& gterms, int64_t B, hipStream_t st) {
  // sized for the [B] part; the (rare) rescale walks the gradient with at least 1024 blocks
  int64_t blocks = (B + kBlock - 1) / kBlock;
  const int64_t wide = (items + kBlock - 1) / kBlock;
  if (grad && blocks < 1024) blocks = wide < 1024 ? (wide > blocks ? wide : blocks) : 1024;
  const int grid = (int)(blocks < 1 ? 1 : (blocks < 4096 ? blocks : 4096));
  hipLaunchKernelGGL((token_elbo_bwd_kernel<T, V>), dim3(grid), dim3(kBlock), 0, st, (const T*)gnll, (const T*)gloss,
                     (const T*)gelbo, gm, gmeans_dtype, kl_beta, inv_count, grow, (T*)grad, items, gterms, B);
}

}  // namespace vae

using namespace vae;

extern "C" {

int vae_token_nll_elbo_terms_fwd(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, int64_t len,
                                 const void* kld, const void* add, const void* mi, int terms_dtype, float kl_beta,
                                 float inv_count, float* logp, float* stats, void* glogits, void* nll, void* loss,
                                 void* elbo, float* means, void* loss_mean, void* other_means, int mean_dtype,
                                 float* workspace, void* scratch, int64_t B, int64_t V, int dtype, vae_stream_t stream) {
  if (B < 0 || len < 0 || V < 1 || V > VAE_MAX_ROW || (B * len > 1 && row_stride < V) || !type_ok(dtype) ||
      ((kld || add || mi) && !type_ok(terms_dtype)) || ((loss_mean || other_means) && !type_ok(mean_dtype)))
    return VAE_ERR_ARG;
  if (B == 0) return VAE_OK;
  const int64_t N = B * len;
  if ((loss == nullptr) != (elbo == nullptr) || (!nll && !loss) || (loss && !means)) return VAE_ERR_ARG;
  if (N > 0 && (!logits || !tokens || (token_bytes != 4 && token_bytes != 8) || !logp || !stats ||
                (vae_token_scratch_bytes(N, V, 0, dtype) && !scratch)))
    return VAE_ERR_ARG;
  int rc = VAE_OK;
  if (N > 0)
    rc = glogits ? token_nll_grad(logits, row_stride, tokens, token_bytes, logp, stats, glogits, inv_count, scratch, N, V,
                                  dtype, (hipStream_t)stream)
                 : vae_token_logp_fwd(logits, row_stride, tokens, token_bytes, logp, nullptr, stats, nullptr, nullptr, 0,
                                      scratch, N, V, dtype, stream);
  if (rc != VAE_OK) return rc;
  const MeansTo to = {loss_mean, other_means, mean_dtype};
  const Terms terms = {kld, add, mi, terms_dtype};
  int G = 1;
  while (G < 64 && G < len) G <<= 1;
  const int64_t blocks = (B + kBlock / G - 1) / (kBlock / G);
  // Without the means nothing is left to add up: as many blocks as there are samples for.  With them a second launch adds
  // the blocks up, unless one large block holds the samples side by side: 16 x 784 tokens 7.6 us with the rows' launch, 9.4
  // with a second one (two turns of it would gain nothing: 32 x 784 10.1, 9.7)
  const int64_t most = loss ? kElboBlocks : kMaxGrid;
  const bool one = loss && blocks > 1 && B <= kOneBlock / G;
  const int grid = one ? 1 : (int)(blocks < most ? blocks : most);
#define VAE_ELBO_FWD(BT)                                                                                                \
  hipLaunchKernelGGL((token_elbo_fwd_kernel<T, BT>), dim3(grid), dim3(BT), 0, (hipStream_t)stream, logp, len,            \
                     terms, kl_beta, inv_count, (T*)nll, (T*)loss, (T*)elbo, means, to, workspace, B, G)
  VAE_BY_TYPE(dtype, if (one) VAE_ELBO_FWD(kOneBlock); else VAE_ELBO_FWD(kBlock));
#undef VAE_ELBO_FWD
  if (loss && grid > 1)
    hipLaunchKernelGGL(token_elbo_means_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, means, grid, inv_count,
                       to, workspace);
  return launched();
}

int vae_token_nll_elbo_fwd(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, int64_t len,
                           const void* kld, const void* add, const void* mi, float kl_beta, float inv_count, float* logp,
                           float* stats, void* glogits, void* nll, void* loss, void* elbo, float* means, void* loss_mean,
                           void* other_means, int mean_dtype, float* workspace, void* scratch, int64_t B, int64_t V,
                           int dtype, vae_stream_t stream) {
  return vae_token_nll_elbo_terms_fwd(logits, row_stride, tokens, token_bytes, len, kld, add, mi, dtype, kl_beta, inv_count,
                                      logp, stats, glogits, nll, loss, elbo, means, loss_mean, other_means, mean_dtype,
                                      workspace, scratch, B, V, dtype, stream);
}

int vae_token_nll_elbo_terms_bwd(const void* gnll, const void* gloss, const void* gelbo, const void* const* gmeans,
                                 int gmeans_dtype, float kl_beta, float inv_count, float* grow, void* grad, int64_t n,
                                 void* gkld, void* gadd, void* gmi, int terms_dtype, int64_t B, int dtype,
                                 vae_stream_t stream) {
  if (B < 0 || n < 0 || !type_ok(dtype) || !type_ok(gmeans_dtype) || ((gkld || gadd || gmi) && !type_ok(terms_dtype)))
    return VAE_ERR_ARG;
  if (grad && (gnll || gloss || gelbo)) return VAE_ERR_ARG;
  if (B == 0 && (n == 0 || !grad)) return VAE_OK;
  Scalars6 gm = {};
  if (gmeans)
    for (int k = 0; k < 6; ++k) gm.p[k] = gmeans[k];
  const GradTerms gterms = {gkld, gadd, gmi, terms_dtype};
  VAE_BY_TYPE(dtype, constexpr int VN = VecOf<T>::n;
              if (n % VN == 0 && aligned16(grad))
                elbo_bwd_launch<T, VN>(gnll, gloss, gelbo, gm, gmeans_dtype, kl_beta, inv_count, grow, grad, n / VN, gterms,
                                       B, (hipStream_t)stream);
              else elbo_bwd_launch<T, 1>(gnll, gloss, gelbo, gm, gmeans_dtype, kl_beta, inv_count, grow, grad, n, gterms, B,
                                         (hipStream_t)stream));
  return launched();
}

int vae_token_nll_elbo_bwd(const void* gnll, const void* gloss, const void* gelbo, const void* const* gmeans,
                           int gmeans_dtype, float kl_beta, float inv_count, float* grow, void* grad, int64_t n,
                           void* gkld, void* gadd, void* gmi, int64_t B, int dtype, vae_stream_t stream) {
  return vae_token_nll_elbo_terms_bwd(gnll, gloss, gelbo, gmeans, gmeans_dtype, kl_beta, inv_count, grow, grad, n, gkld,
                                      gadd, gmi, dtype, B, dtype, stream);
}

int vae_grad_scale(void* buf, const float* factor, int64_t n, int dtype, vae_stream_t stream) {
  if (n < 0) return VAE_ERR_ARG;
  if (n == 0) return type_ok(dtype) ? VAE_OK : VAE_ERR_ARG;
  if (!buf || !factor) return VAE_ERR_ARG;
  const void* g[6] = {factor, nullptr, nullptr, nullptr, nullptr, nullptr};
  return vae_token_nll_elbo_bwd(nullptr, nullptr, nullptr, g, VAE_F32, 0.f, 0.f, nullptr, buf, n, nullptr, nullptr,
                                nullptr, 0, dtype, stream);
}

int vae_row_sums(const float* rows, float scale, void* out, int64_t B, int64_t len, int dtype, vae_stream_t stream) {
  if (B < 0 || len < 0 || !type_ok(dtype)) return VAE_ERR_ARG;
  if (B == 0) return VAE_OK;
  if (!out || (len > 0 && !rows)) return VAE_ERR_ARG;
  const int grid = (int)(B < kMaxGrid ? B : kMaxGrid);
  VAE_BY_TYPE(dtype, if (len > 4096) hipLaunchKernelGGL((row_sums_kernel<T, 1024>), dim3(grid), dim3(1024), 0,
                                                        (hipStream_t)stream, rows, scale, (T*)out, B, len);
              else hipLaunchKernelGGL((row_sums_kernel<T, kBlock>), dim3(grid), dim3(kBlock), 0, (hipStream_t)stream, rows,
                                      scale, (T*)out, B, len));
  return launched();
}

}  // extern "C"
