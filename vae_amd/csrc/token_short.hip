// Short rows of logits (at most 256 vectors: 2048 16-bit or 1024 fp32 entries, 256 of either where a row is not aligned):
// a row is held by a group of G lanes, several rows to a wave, and everything that is asked of it -- log prob,
// entropy, alternatives, gradient -- comes from those registers.  The backward pass recomputes the row's statistics: they
// cost less than reading them.  Formulas and the conventions for masks: token_row.hpp.
#include "token_row.hpp"

namespace vae {

template <typename T, int VN, int U, bool ENT>
__global__ __launch_bounds__(kBlock) void token_short_kernel(ShortArgs a, int G, int64_t tiles) {
  const int rpb = kBlock / G, sub = threadIdx.x % G, rloc = threadIdx.x / G;
  const int nvec = a.V / VN;
  const bool nts = nt_stores((int64_t)a.N * a.V * (int64_t)sizeof(T));
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row = tile * rpb + rloc;
    const bool live = row < a.N;
    const int64_t r = live ? row : a.N - 1;
    const T* x = (const T*)a.logits + r * a.row_stride;
    const int64_t tok = a.tokens ? load_id(a.tokens, a.token_bytes, r) : 0;
    const bool pad = tok < 0 || !live;
    float v[U][VN];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = sub + u * G;
      if (j < nvec && !pad) {
        load_vec<T, VN>(x + j * VN, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VN; ++i) v[u][i] = -INFINITY;
      }
    }
    float m = kLowest;
#pragma unroll
    for (int u = 0; u < U; ++u) m = vec_max(v[u], m);
    m = group_max(m, G);
    float s = 0.f, t = 0.f, e[U][VN];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const float d = (v[u][i] - m) * kLog2e;
        e[u][i] = exp2_raw(d);
        s += e[u][i];
        if constexpr (ENT) t = __builtin_fmaf(max_raw(d, -300.f), e[u][i], t);
      }
    s = group_sum(s, G);
    float h = 0.f;
    if constexpr (ENT) {
      t = group_sum(t, G);
      h = s == 0.f ? 0.f : kLn2 * (log2f(s) - t / s);
    }
    if (sub == 0 && live) {
      if (a.logp) a.logp[row] = pad ? 0.f : (tok < a.V ? row_log_prob(to_f32(x[tok]), m, s, 1.0f) : nan_f());
      if constexpr (ENT) {
        if (a.entropy) a.entropy[row] = h;
      }
      if (a.stats) {
        a.stats[2 * row] = m;
        a.stats[2 * row + 1] = s;
      }
    }
    if (a.top_k) {
      uint64_t last = ~0ull;
      for (int k = 0; k < a.top_k; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (sub + u * G < nvec)
#pragma unroll
            for (int i = 0; i < VN; ++i) {
              const uint64_t key = order_key(v[u][i], (uint32_t)((sub + u * G) * VN + i));
              best = key < last && key > best ? key : best;
            }
        for (int o = G >> 1; o >= 1; o >>= 1) {
          const uint64_t w = __shfl_xor(best, o, 64);
          best = w > best ? w : best;
        }
        last = best;
        if (sub == 0 && live) {
          a.top_logp[row * a.top_k + k] = pad ? -INFINITY : (best ? row_log_prob(key_value(best), m, s, 1.0f) : nan_f());
          a.top_ids[row * a.top_k + k] = pad || !best ? -1 : key_index(best);
        }
      }
    }
    if (!a.glogits || !live) continue;
    const bool zero = pad || s == 0.f;
    float gt = a.tokens ? (a.glogp ? a.glogp[row / a.rows_per_g] * a.g_scale : a.g_scale) : 0.f;
    if (tok >= a.V && (!a.glogp || a.g_scale != 0.f)) gt = nan_f();
    float sum = gt;
    for (int k = 0; k < a.gtop_k; ++k) sum += a.gtop[row * a.gtop_k + k];
    const float inv = 1.0f / s;
    float B = 0.f;
    if constexpr (ENT) {
      const float gh = a.gentropy ? a.gentropy[row] : 0.f;
      sum += gh * (h - kLn2 * log2f(s));
      B = -gh * kLn2 * inv;
    }
    const float A = -sum * inv;
    T* gx = (T*)a.glogits + row * (int64_t)a.V;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VN; ++i)
        e[u][i] *= ENT ? __builtin_fmaf(B, max_raw((v[u][i] - m) * kLog2e, -300.f), A) : A;
    auto add = [&](int64_t id, float g) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = id - (sub + u * G) * VN;
#pragma unroll
        for (int i = 0; i < VN; ++i) e[u][i] += at == i ? g : 0.f;
      }
    };
    if (a.tokens) add(tok < a.V ? tok : -1, gt);
    for (int k = 0; k < a.gtop_k; ++k) add(a.gtop_ids[row * a.gtop_k + k], a.gtop[row * a.gtop_k + k]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = sub + u * G;
      if (j < nvec) {
        if (zero)
#pragma unroll
          for (int i = 0; i < VN; ++i) e[u][i] = 0.f;
        store_vec<T, VN>(nts, gx + j * VN, e[u]);
      }
    }
  }
}

template <typename T, int VN, bool ENT>
static int short_launch(const ShortArgs& a, const RowGeom& g, hipStream_t st) {
  VAE_SWITCH_U(g.U, hipLaunchKernelGGL((token_short_kernel<T, VN, U, ENT>), dim3(g.grid), dim3(kBlock), 0, st, a, g.G,
                                       g.tiles));
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
}
template <typename T, int VN>
static int short_kind(const ShortArgs& a, const RowGeom& g, hipStream_t st) {
  return a.entropy || a.gentropy ? short_launch<T, VN, true>(a, g, st) : short_launch<T, VN, false>(a, g, st);
}

bool short_rows(const ShortArgs& a, int dtype, hipStream_t st, int* rc) {
  const int64_t vn = dtype == VAE_F32 ? 4 : 8;
  const bool vec = a.V % vn == 0 && (a.N <= 1 || a.row_stride % vn == 0) && aligned16(a.logits) &&
                   (!a.glogits || aligned16(a.glogits));
  const int64_t nvec = vec ? a.V / vn : a.V;
  RowGeom g;
  if (nvec > 4 * 64 || !row_geom_resident(a.N, nvec, kGridStream, &g)) return false;
  VAE_BY_TYPE(dtype, *rc = vec ? short_kind<T, VecOf<T>::n>(a, g, st) : short_kind<T, 1>(a, g, st));
  return true;
}

}  // namespace vae
