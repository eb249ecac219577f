// Short rows of logits (up to 1024 entries, 256 where rows are not aligned; see `takes`): a row is held by a group of G
// lanes, several rows to a wave, and everything that is asked of it -- log prob, entropy, alternatives, gradient -- comes
// from those registers.  The backward pass recomputes the row's statistics: they cost less than reading them.  Bound by
// memory: loss and gradient of 200704 x 256 bf16 43 us (4.8 TB/s read + written), 65536 x 1024 fp32 87 us (6.2 TB/s).
// Formulas and the conventions for masks: token_row.hpp.
#include "token_row.hpp"

namespace vae {

enum { kEnt = 1, kTop = 2, kGrad = 4 };   // what a kernel forms beside log prob and statistics

template <typename T, int VN, int U, int WHAT>
__global__ __launch_bounds__(kBlock) void token_short_kernel(ShortArgs a, int log_g, int64_t tiles) {
  constexpr bool ENT = WHAT & kEnt, TOP = WHAT & kTop, GRAD = WHAT & kGrad;
  const int G = 1 << log_g;
  const int sub = threadIdx.x & (G - 1), rloc = threadIdx.x >> log_g;
  const int nvec = a.V / VN;
  const bool nts = nt_stores((int64_t)a.N * a.V * (int64_t)sizeof(T));
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row = (tile << (8 - log_g)) + rloc;     // kBlock / G rows a tile
    const bool live = row < a.N;
    const int64_t r = live ? row : a.N - 1;
    const T* x = (const T*)a.logits + r * a.row_stride;
    const int64_t tok64 = a.tokens ? load_id(a.tokens, a.token_bytes, r) : 0;
    const bool pad = tok64 < 0 || !live, beyond = tok64 >= a.V;
    const int tok = pad || beyond ? -1 : (int)tok64;
    const float token_logit = a.logp && tok >= 0 ? to_f32(x[tok]) : 0.f;
    float v[U][VN];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = sub + (u << log_g);
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
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const float d = (v[u][i] - m) * kLog2e;
        const float ev = exp2_raw(d);
        s += ev;
        if constexpr (ENT) t = __builtin_fmaf(max_raw(d, -300.f), ev, t);
        if constexpr (GRAD) e[u][i] = ev;
      }
      __builtin_amdgcn_sched_barrier(0);   // vector by vector: fewer registers
    }
    s = group_sum(s, G);
    const float ls = log2f(s);
    float h = 0.f;
    if constexpr (ENT) {
      t = group_sum(t, G);
      h = s == 0.f ? 0.f : kLn2 * (ls - t / s);
    }
    if (sub == 0 && live) {
      if (a.logp)
        a.logp[row] = pad ? 0.f : (beyond ? nan_f() : (s == 0.f ? -INFINITY : token_logit - m - kLn2 * ls));
      if constexpr (ENT) {
        if (a.entropy) a.entropy[row] = h;
      }
      if (a.stats) {
        a.stats[2 * row] = m;
        a.stats[2 * row + 1] = s;
      }
    }
    if constexpr (TOP) {
      uint64_t last = ~0ull;
      for (int k = 0; k < a.top_k; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (sub + (u << log_g) < nvec)
#pragma unroll
            for (int i = 0; i < VN; ++i) {
              const uint64_t key = order_key(v[u][i], (uint32_t)((sub + (u << log_g)) * VN + i));
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
    if constexpr (GRAD) {
      if (!live) continue;
      float gt = 0.f;
      if (a.tokens) {
        gt = a.g_scale;
        if (a.glogp) {
          int64_t at = row;
          if (a.rows_per_g != 1)   // a 64-bit division costs as much as the row
            at = (a.N | a.rows_per_g) >> 32 ? row / a.rows_per_g
                                            : (int64_t)((uint32_t)row / (uint32_t)a.rows_per_g);
          gt *= a.glogp[at];
        }
      }
      float sum = gt;
      for (int k = 0; k < a.gtop_k; ++k) sum += a.gtop[row * a.gtop_k + k];
      const float inv = 1.0f / s;
      float B = 0.f;
      if constexpr (ENT) {
        const float gh = a.gentropy[row];
        sum += gh * (h - kLn2 * ls);
        B = -gh * kLn2 * inv;
      }
      const float A = -sum * inv;
      const bool bad = beyond && (!a.glogp || a.g_scale != 0.f);   // the gradient of its NaN
      const bool fixed = pad || s == 0.f || bad;
      T* gx = (T*)a.glogits + row * (int64_t)a.V;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = sub + (u << log_g);
        float o[VN];
#pragma unroll
        for (int i = 0; i < VN; ++i)
          o[i] = e[u][i] * (ENT ? __builtin_fmaf(B, max_raw((v[u][i] - m) * kLog2e, -300.f), A) : A);
        auto add = [&](int id, float g) {
          const int at = id - j * VN;
          if (at >= 0 && at < VN)
#pragma unroll
            for (int i = 0; i < VN; ++i) o[i] += at == i ? g : 0.f;
        };
        add(tok, gt);
        for (int k = 0; k < a.gtop_k; ++k) add((int)a.gtop_ids[row * a.gtop_k + k], a.gtop[row * a.gtop_k + k]);
        if (j < nvec) {
          if (fixed)
#pragma unroll
            for (int i = 0; i < VN; ++i) o[i] = bad ? nan_f() : 0.f;
          store_vec<T, VN>(nts, gx + j * VN, o);
        }
      }
    }
  }
}

template <typename T, int VN, int WHAT>
static int short_launch(const ShortArgs& a, const RowGeom& g, hipStream_t st) {
  const int log_g = __builtin_ctz(g.G);
  VAE_SWITCH_U(g.U, hipLaunchKernelGGL((token_short_kernel<T, VN, U, WHAT>), dim3(g.grid), dim3(kBlock), 0, st, a, log_g,
                                       g.tiles));
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
}
template <typename T, int VN>
static int short_kind(const ShortArgs& a, const RowGeom& g, hipStream_t st) {
  if (a.glogits) return a.gentropy ? short_launch<T, VN, kGrad | kEnt>(a, g, st) : short_launch<T, VN, kGrad>(a, g, st);
  if (a.top_k) return a.entropy ? short_launch<T, VN, kTop | kEnt>(a, g, st) : short_launch<T, VN, kTop>(a, g, st);
  return a.entropy ? short_launch<T, VN, kEnt>(a, g, st) : short_launch<T, VN, 0>(a, g, st);
}

// Which rows these kernels take, against the long ones (token.hip, token_grad.hip) for 65536 rows, in us:
//   log prob of 256 bf16 9.3 / 27, 1024 bf16 29 / 38, 1024 fp32 41 / 42, but 2000 bf16 55 / 62 and 2048 bf16 54 / 49;
//   loss and gradient 256 bf16 17 / 56, 1024 bf16 58 / 78, 1024 fp32 93 / 107, 2048 bf16 104 / 96: up to 1024 entries.
//   Entropy's gradient holds value and exponential: 512 bf16 36 / 40, but 1024 bf16 65 / 54 (8 registers a vector each).
//   Alternatives cost a turn over the registers each: 256 bf16 k = 8 44 / 73, k = 20 79 / 84; 512 bf16 k = 4 57 / 68,
//   k = 8 80 / 75; 1024 bf16 k = 4 111 / 83: while k V < 4096; beyond 48 of them the long kernel's bound gives way (k = 64:
//   256 bf16 213 / 486, 512 bf16 425 / 470, 1024 bf16 860 / 650).
static bool takes(const ShortArgs& a, bool wide) {
  if (a.V > 1024 || (a.glogits && a.gentropy && !wide && a.V > 512)) return false;
  return (int64_t)a.top_k * a.V < 4096 || (a.top_k > 48 && a.V <= 512);
}

bool short_rows(const ShortArgs& a, int dtype, hipStream_t st, int* rc) {
  const int64_t vn = dtype == VAE_F32 ? 4 : 8;
  const bool vec = a.V % vn == 0 && (a.N <= 1 || a.row_stride % vn == 0) && aligned16(a.logits) &&
                   (!a.glogits || aligned16(a.glogits));
  const int64_t nvec = vec ? a.V / vn : a.V;
  RowGeom g;
  if (nvec > 4 * 64 || !takes(a, dtype == VAE_F32) || !row_geom_resident(a.N, nvec, kGridStream, &g)) return false;
  VAE_BY_TYPE(dtype, *rc = vec ? short_kind<T, VecOf<T>::n>(a, g, st) : short_kind<T, 1>(a, g, st));
  return true;
}

}  // namespace vae
