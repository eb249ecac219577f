// Gradients with respect to rows of logits [N, V]: of log probs, entropy and alternatives (token_logp_bwd), of the
// distillation KL (distill_bwd), and both losses together with their gradient in one pass (token_nll_fused,
// distill_fwd with glogits).  Formulas and the conventions for masks: token_row.hpp.
//
// Every one of them is   g_j = e_j (A + B d_j) + sum over a few entries (id, g) with id = j,   d = (x - m) c, e = 2^d:
//   tokens:   A = -(sum_i g_i + g_H (H - ln s)) / s,  B = -g_H ln2 / s,  entries: the token and the alternatives
//   teacher:  A = w / (tau s),  B = 0,  entries: (id_k, -w q_k / tau)
// The entries are owned by the thread whose vector holds them and added before the vector is stored: no atomics on the
// gradient, no second write, one rounding.
#include "token_row.hpp"

namespace vae {

// A piece's entries in LDS: each thread's own in a list.  Entries of one id are merged first, in entry order, so what
// a gradient element receives does not depend on the order of the list.
constexpr int kMaxEntries = VAE_MAX_TEACHER;
template <int BT>
struct Entries {
  static constexpr int R = (kMaxEntries + BT - 1) / BT;
  int head[BT];
  int next[kMaxEntries], id[kMaxEntries];
  float g[kMaxEntries];

  // id[0..n), g[0..n) have been written by the workgroup (id < 0: none)
  template <typename T, int VN>
  __device__ __forceinline__ void link(int n, const RowCut<T, VN>& cut, int v0, int v1) {
    int own[R];
    float sum[R];
    head[threadIdx.x] = -1;
    lds_barrier();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = threadIdx.x + r * BT;
      own[r] = k < n ? id[k] : -1;
      sum[r] = 0.f;
      if (own[r] >= 0) {
        bool first = true;
        for (int q = 0; q < n; ++q)
          if (id[q] == own[r]) {
            first &= q >= k;
            sum[r] += g[q];
          }
        if (!first) own[r] = -1;
      }
    }
    lds_barrier();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = threadIdx.x + r * BT;
      if (own[r] < 0) continue;
      g[k] = sum[r];
      const int off = own[r] - cut.head;
      int owner = -1;
      if (off < 0) owner = own[r];                                      // RowCut::edge
      else if (off >= cut.nvec * VN) owner = 16 + off - cut.nvec * VN;
      else if (off / VN >= v0 && off / VN < v1) owner = (off / VN - v0) % BT;
      if (owner >= 0) next[k] = atomicExch(&head[owner], k);
    }
    lds_barrier();
  }
};

// What a thread adds to its elements: one entry known to all (ONE), or the workgroup's lists.
template <typename T, int VN, int BT, bool LIST>
struct Adds {
  const Entries<BT>* lds;
  int one_id;        // -1: none
  float one_g;
  uint32_t mask;     // bit u: the thread's u-th vector of the piece holds an entry (at most 32 vectors)

  __device__ __forceinline__ void prepare(const RowCut<T, VN>& cut, int v0, int v1) {
    mask = 0;
    auto note = [&](int id) {
      const int off = id - cut.head, vec = off / VN;
      if (off >= 0 && vec < cut.nvec && vec >= v0 && vec < v1 && (vec - v0) % BT == (int)threadIdx.x)
        mask |= 1u << ((vec - v0) / BT);
    };
    if constexpr (LIST) {
      for (int k = lds->head[threadIdx.x]; k >= 0; k = lds->next[k]) note(lds->id[k]);
    } else if (one_id >= 0) {
      note(one_id);
    }
  }
  template <int W>
  __device__ __forceinline__ void to(int index, float (&v)[W]) const {
    auto add = [&](int id, float g) {
      const int e = id - index;
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] += e == i ? g : 0.f;   // as a select: v stays in registers
    };
    if constexpr (LIST) {
      for (int k = lds->head[threadIdx.x]; k >= 0; k = lds->next[k]) add(lds->id[k], lds->g[k]);
    } else {
      add(one_id, one_g);
    }
  }
};

struct GradArgs {
  const void* logits;
  int64_t row_stride;
  void* glogits;
  int64_t N;
  int V, parts;
  bool nts;
  float scale2, inv_tau;
  const float* stats_in;
  // tokens
  const void* tokens;
  int token_bytes;
  const float *entropy, *glogp;
  int64_t rows_per_g;
  float g_scale;
  const float *gentropy, *gtop;
  const int64_t* top_ids;
  int top_k;
  // teacher
  TeacherArgs teacher;
  const float *gkl, *gmean;
  float mean_scale;
  // fused
  float *out, *stats_out;            // logp or kl, and the statistics
};

// A thread's U vectors of a piece of a row, v0 + tid, v0 + tid + BT, ...  `nvec`: vectors of the piece (a piece is at
// most U * BT vectors, 1 MiB).
template <typename T, int VN, int BT, int U>
struct Piece {
  typedef Packet<T, VN> P;
  P p[U];
  const Buffer in, out;
  const int nvec, byte;

  __device__ __forceinline__ Piece(const T* x, T* gx, const RowCut<T, VN>& cut, int v0, int nvec_)
      : in(x + cut.index(v0), nvec_ * P::kBytes), out(gx + cut.index(v0), nvec_ * P::kBytes), nvec(nvec_),
        byte((int)threadIdx.x * P::kBytes) {}
  __device__ __forceinline__ bool any(int u) const { return u * BT < nvec; }   // the same for all threads
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int u = 0; u < U; ++u) p[u].load(in, byte, u * BT * P::kBytes);
  }
  __device__ __forceinline__ void mask() {       // what is not there counts as masked out
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((u + 1) * BT > nvec && (int)threadIdx.x + u * BT >= nvec) p[u].set_masked();
  }
  __device__ __forceinline__ void store(bool nts, int u, const float (&v)[VN]) const {
    P::store(out, nts, byte, u * BT * P::kBytes, v);
  }
  __device__ __forceinline__ void fill(bool nts, float value) const {
    float v[VN];
#pragma unroll
    for (int i = 0; i < VN; ++i) v[i] = value;
#pragma unroll
    for (int u = 0; u < U; ++u) store(nts, u, v);
  }
};

// ---------------------------------------------------------------------------------------------------------------
// from given statistics: one read, one write.  A workgroup takes one piece of U vectors a thread, all loads in front of
// all stores: in a loop the loads of a turn wait for the stores of the turn before it (4096 x 32768 bf16: 153 us with
// a loop over U = 4, see bwd_launch for what one piece takes).
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int VN, int BT, int U, bool ENT, bool LIST, bool DIST>
__global__ __launch_bounds__(BT) void token_bwd_kernel(GradArgs a) {
  __shared__ struct {
    Entries<BT> entries[LIST ? 1 : 0];
    TeacherRow<BT> teacher[DIST ? 1 : 0];
  } lds;
  for (int64_t item = blockIdx.x; item < a.N * a.parts; item += gridDim.x) {
    const int64_t row = a.parts == 1 ? item : item / a.parts;
    const int part = a.parts == 1 ? 0 : (int)(item - row * a.parts);
    const T* x = (const T*)a.logits + row * a.row_stride;
    T* gx = (T*)a.glogits + row * (int64_t)a.V;
    const RowCut<T, VN> cut(x, a.V);
    const int v0 = part * (U * BT);
    const int left = cut.nvec - v0;
    const int v1 = v0 + (left < 0 ? 0 : (left < U * BT ? left : U * BT));
    int ei = cut.edge(threadIdx.x);
    if (ei >= 0 && (ei < cut.head ? part != 0 : part != a.parts - 1)) ei = -1;
    Piece<T, VN, BT, U> piece(x, gx, cut, v0, v1 - v0);
    const float m = a.stats_in[2 * row], s = a.stats_in[2 * row + 1];
    const int64_t tok = !DIST && a.tokens ? load_id(a.tokens, a.token_bytes, row) : 0;
    if (tok < 0 || s == 0.f) {
      piece.fill(a.nts, 0.f);
      if (ei >= 0) gx[ei] = from_f32<T>(0.f);
      continue;
    }
    piece.load();
    const float edge = ei >= 0 ? to_f32(x[ei]) : 0.f;
    Adds<T, VN, BT, LIST> adds;
    if constexpr (LIST) adds.lds = lds.entries;
    float A, B = 0.f;
    const float inv = 1.0f / s;
    if constexpr (DIST) {
      lds.teacher[0].load(a.teacher, row, a.V, a.inv_tau, a.scale2);   // an id beyond the vocabulary: s is NaN
      const float g0 = a.gmean ? a.gmean[0] * a.mean_scale : (a.gkl ? 0.f : a.mean_scale);
      const float w = ((a.gkl ? a.gkl[row] : 0.f) + g0) * a.inv_tau;
      A = w * inv;
      for (int k = threadIdx.x; k < a.teacher.K; k += BT) {
        lds.entries[0].id[k] = lds.teacher[0].id[k];
        lds.entries[0].g[k] = -w * lds.teacher[0].q[k];
      }
    } else {
      float gt = a.tokens ? (a.glogp ? a.glogp[row / a.rows_per_g] * a.g_scale : a.g_scale) : 0.f;
      const bool inside = a.tokens && tok < a.V;
      if (tok >= a.V && (!a.glogp || a.g_scale != 0.f)) gt = nan_f();
      float sum = gt;
      adds.one_id = inside ? (int)tok : -1;
      adds.one_g = gt;
      if constexpr (LIST) {
        for (int k = 0; k < a.top_k; ++k) sum += a.gtop[row * a.top_k + k];
        lds_barrier();  // the row before this one has been read
        for (int k = threadIdx.x; k <= a.top_k; k += BT) {
          lds.entries[0].id[k] = k == 0 ? adds.one_id : (int)a.top_ids[row * a.top_k + k - 1];
          lds.entries[0].g[k] = k == 0 ? gt : a.gtop[row * a.top_k + k - 1];
        }
      }
      if constexpr (ENT) {
        const float gh = a.gentropy[row];
        sum += gh * (a.entropy[row] - kLn2 * log2f(s));
        B = -gh * kLn2 * inv;
      }
      A = -sum * inv;
    }
    if constexpr (LIST) lds.entries[0].template link<T, VN>(DIST ? a.teacher.K : a.top_k + 1, cut, v0, v1);
    adds.prepare(cut, v0, v1);
    auto grad = [&](float v) {
      const float d = (v - m) * a.scale2;
      const float e = exp2_raw(d);
      return ENT ? e * __builtin_fmaf(B, max_raw(d, -300.f), A) : e * A;
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (piece.any(u)) {
        float v[VN];
        piece.p[u].get(v);
#pragma unroll
        for (int i = 0; i < VN; ++i) v[i] = grad(v[i]);
        if (adds.mask >> u & 1u) adds.to(cut.index(v0 + u * BT + (int)threadIdx.x), v);
        piece.store(a.nts, u, v);
      }
    if (ei >= 0) {
      float v[1] = {grad(edge)};
      adds.to(ei, v);
      gx[ei] = from_f32<T>(v[0]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// loss and gradient in one pass: a workgroup holds its row in registers, U vectors a thread.
//   KEEP: every element's exponential against the thread's own maximum, in float32: one exponential an element, the
//         gradient is a product.  8 registers a 16-bit vector, 4 an fp32 one.
//   else: the packets as they were read, 4 registers a vector whatever the type; the exponentials are formed twice.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int BT, int U, bool KEEP, bool DIST>
__global__ __launch_bounds__(BT) void token_fused_kernel(GradArgs a) {
  constexpr int VN = VecOf<T>::n;
  __shared__ struct {
    Entries<BT> entries[DIST ? 1 : 0];
    TeacherRow<BT> teacher[DIST ? 1 : 0];
  } lds;
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* x = (const T*)a.logits + row * a.row_stride;
    T* gx = (T*)a.glogits + row * (int64_t)a.V;
    const RowCut<T, VN> cut(x, a.V);
    const int ei = cut.edge(threadIdx.x);
    Piece<T, VN, BT, U> piece(x, gx, cut, 0, cut.nvec);
    int64_t tok = 0;
    int state = kRowFine;
    typename TeacherRow<BT>::Mine mine;
    if constexpr (DIST) {
      if (!TeacherRow<BT>::fetch(mine, a.teacher, row, a.V)) state = kRowEmpty;
    } else {
      tok = load_id(a.tokens, a.token_bytes, row);
      state = tok < 0 ? kRowEmpty : (tok >= a.V ? kRowBad : kRowFine);
    }
    if (state != kRowFine) {
      const float v = state == kRowEmpty ? 0.f : nan_f();
      piece.fill(a.nts, v);
      if (ei >= 0) gx[ei] = from_f32<T>(v);
      if (threadIdx.x == 0) {
        a.out[row] = v;
        a.stats_out[2 * row] = 0.f;
        a.stats_out[2 * row + 1] = v;
      }
      continue;
    }
    piece.load();
    const float edge = ei >= 0 ? to_f32(x[ei]) : -INFINITY;
    Adds<T, VN, BT, DIST> adds;
    const float w = DIST ? a.mean_scale * a.inv_tau : a.g_scale;   // of p; the entries have the other sign
    if constexpr (DIST) {
      // while the row is on its way
      state = lds.teacher[0].finish(mine, a.teacher, a.V, a.inv_tau, a.scale2);
      for (int k = threadIdx.x; k < a.teacher.K; k += BT) {
        const int id = lds.teacher[0].id[k];
        lds.teacher[0].x[k] = id >= 0 ? to_f32(x[id]) : 0.f;
        lds.entries[0].id[k] = id;
        lds.entries[0].g[k] = -w * lds.teacher[0].q[k];
      }
      adds.lds = lds.entries;
      lds.entries[0].template link<T, VN>(a.teacher.K, cut, 0, cut.nvec);
    } else {
      adds.one_id = (int)tok;
      adds.one_g = -w;
    }
    adds.prepare(cut, 0, cut.nvec);
    piece.mask();
    float mt = max_raw(edge, kLowest);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (piece.any(u)) {
        float v[VN];
        piece.p[u].get(v);
        mt = vec_max(v, mt);
      }
    float e[KEEP ? U : 1][VN];
    float s = exp2_raw((edge - mt) * a.scale2);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (piece.any(u)) {
        asm volatile("" : "+v"(piece.p[u].raw));   // unpack again: the packets, not their elements, stay in registers
        float v[VN];
        piece.p[u].get(v);
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const float ev = exp2_raw((v[i] - mt) * a.scale2);
          s += ev;
          if constexpr (KEEP) e[u][i] = ev;
        }
      }
    const float m = block_max<BT>(mt);
    float f = exp2_raw((mt - m) * a.scale2);       // from the thread's maximum to the row's
    s = block_sum<BT>(s * f);
    if (DIST && state == kRowBad) s = nan_f();
    if constexpr (DIST) {
      float kl = 0.f;
      for (int k = threadIdx.x; k < a.teacher.K; k += BT)
        if (lds.teacher[0].id[k] >= 0)
          kl += lds.teacher[0].q[k] * (lds.teacher[0].logq[k] - row_log_prob(lds.teacher[0].x[k], m, s, a.inv_tau));
      kl = block_sum<BT>(kl);
      if (threadIdx.x == 0) a.out[row] = state == kRowBad ? nan_f() : kl;
    } else if (threadIdx.x == 0) {
      a.out[row] = row_log_prob(to_f32(x[tok]), m, s, 1.0f);
    }
    if (threadIdx.x == 0) {
      a.stats_out[2 * row] = m;
      a.stats_out[2 * row + 1] = s;
    }
    if (s == 0.f) {
      piece.fill(a.nts, 0.f);
      if (ei >= 0) gx[ei] = from_f32<T>(0.f);
      continue;
    }
    const float A = w / s;
    f *= A;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (piece.any(u)) {
        float v[VN];
        if constexpr (KEEP) {
#pragma unroll
          for (int i = 0; i < VN; ++i) v[i] = f * e[u][i];
        } else {
          asm volatile("" : "+v"(piece.p[u].raw));
          piece.p[u].get(v);
#pragma unroll
          for (int i = 0; i < VN; ++i) v[i] = A * exp2_raw((v[i] - m) * a.scale2);
        }
        if (adds.mask >> u & 1u) adds.to(cut.index(u * BT + (int)threadIdx.x), v);
        piece.store(a.nts, u, v);
      }
    if (ei >= 0) {
      float v[1] = {A * exp2_raw((edge - m) * a.scale2)};
      adds.to(ei, v);
      gx[ei] = from_f32<T>(v[0]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------
static bool type_ok(int d) { return d == VAE_F32 || d == VAE_BF16 || d == VAE_F16; }
static bool bad_rows(int64_t N, int64_t V, int64_t row_stride, int dtype) {
  return N < 0 || V < 1 || V > VAE_MAX_ROW || (N > 1 && row_stride < V) || !type_ok(dtype);
}
static int launched() { return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH; }
static int grid_for(int64_t items) { return (int)(items < kMaxGrid ? items : kMaxGrid); }

// logits and gradient rows start at the same offset from a 16-byte boundary, all of them
template <typename T>
static bool same_phase(const GradArgs& a) {
  const int64_t by = (int64_t)reinterpret_cast<uintptr_t>(a.logits) - (int64_t)reinterpret_cast<uintptr_t>(a.glogits);
  return by % 16 == 0 && (a.N <= 1 || (a.row_stride - a.V) * (int64_t)sizeof(T) % 16 == 0);
}

template <typename T, int VN, int BT, int U, bool ENT, bool LIST, bool DIST>
static int bwd_launch(GradArgs a, hipStream_t st) {
  const int64_t nvec = ((int64_t)a.V + VN - 1) / VN;
  a.parts = (int)((nvec + U * BT - 1) / (U * BT));
  a.nts = (int64_t)sizeof(T) * a.N * a.V >= kNtStoreMinBytes;
  hipLaunchKernelGGL((token_bwd_kernel<T, VN, BT, U, ENT, LIST, DIST>), dim3(grid_for(a.N * a.parts)), dim3(BT), 0, st,
                     a);
  return launched();
}
template <typename T, int VN, bool ENT, bool LIST, bool DIST>
static int bwd_block(const GradArgs& a, hipStream_t st) {
  const int64_t nvec = ((int64_t)a.V + VN - 1) / VN;
  if (nvec <= 256) return bwd_launch<T, VN, 64, 4, ENT, LIST, DIST>(a, st);
  // the entries are prepared once a piece: longer pieces where there are many
  return bwd_launch<T, VN, kBlock, LIST ? 8 : 4, ENT, LIST, DIST>(a, st);
}
template <typename T, int VN, bool DIST>
static int bwd_kind(const GradArgs& a, hipStream_t st) {
  if constexpr (DIST) return bwd_block<T, VN, false, true, true>(a, st);
  else {
    const bool list = a.gtop != nullptr;
    if (a.gentropy) return list ? bwd_block<T, VN, true, true, false>(a, st) : bwd_block<T, VN, true, false, false>(a, st);
    return list ? bwd_block<T, VN, false, true, false>(a, st) : bwd_block<T, VN, false, false, false>(a, st);
  }
}
template <typename T, bool DIST>
static int bwd_type(const GradArgs& a, hipStream_t st) {
  return same_phase<T>(a) ? bwd_kind<T, VecOf<T>::n, DIST>(a, st) : bwd_kind<T, 1, DIST>(a, st);
}

template <typename T, int BT, int U, bool KEEP, bool DIST>
static int fused_launch(GradArgs a, hipStream_t st) {
  a.nts = (int64_t)sizeof(T) * a.N * a.V >= kNtStoreMinBytes;
  hipLaunchKernelGGL((token_fused_kernel<T, BT, U, KEEP, DIST>), dim3(grid_for(a.N)), dim3(BT), 0, st, a);
  return launched();
}
// true when the one-pass kernel takes this call: the row fits a workgroup's registers, and there are rows enough
template <typename T, bool DIST>
static bool fused_type(const GradArgs& a, hipStream_t st, int* rc) {
  constexpr int E = 64 / VecOf<T>::n;    // vectors a thread: 64 elements
  const int64_t nvec = (int64_t)a.V / VecOf<T>::n;
  if (!same_phase<T>(a) || nvec > 16384 || (a.N < 256 && nvec > 4096)) return false;
  if (nvec <= 64 * E) *rc = fused_launch<T, 64, E, true, DIST>(a, st);
  else if (nvec <= 128 * E) *rc = fused_launch<T, 128, E, true, DIST>(a, st);
  else if (nvec <= 256 * E) *rc = fused_launch<T, 256, E, true, DIST>(a, st);
  else if (nvec <= 512 * E) *rc = fused_launch<T, 512, E, true, DIST>(a, st);
  else if (nvec <= 1024 * E) *rc = fused_launch<T, 1024, E, true, DIST>(a, st);
  else *rc = fused_launch<T, 1024, 16, false, DIST>(a, st);
  return true;
}

static bool bad_teacher(const TeacherArgs& t, int64_t N, float temperature) {
  return !type_ok(t.dtype) || t.K < 1 || t.K > VAE_MAX_TEACHER || (N > 1 && (t.stride < t.K || t.id_stride < t.K)) ||
         (t.id_bytes != 4 && t.id_bytes != 8) || !(temperature > 0.f) || !(temperature < INFINITY);
}
static void set_temperature(GradArgs& a, float temperature) {
  a.scale2 = (float)(1.4426950408889634 / (double)temperature);
  a.inv_tau = (float)(1.0 / (double)temperature);
}

}  // namespace vae

using namespace vae;

extern "C" {

int vae_token_logp_bwd(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, const float* stats,
                       const float* entropy, const float* glogp, int64_t rows_per_g, float g_scale,
                       const float* gentropy, const float* gtop, const int64_t* top_ids, int64_t top_k, void* glogits,
                       int64_t N, int64_t V, int dtype, vae_stream_t stream) {
  if (bad_rows(N, V, row_stride, dtype) || top_k < 0 || top_k > VAE_MAX_TOP || rows_per_g < 1) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !stats || !glogits || (tokens && token_bytes != 4 && token_bytes != 8)) return VAE_ERR_ARG;
  if ((gentropy && !entropy) || (top_k > 0 && (!gtop || !top_ids)) || (glogp && !tokens)) return VAE_ERR_ARG;
  int rc = VAE_OK;
  ShortArgs sa = {logits, row_stride, tokens, token_bytes, N, (int)V, nullptr, nullptr, nullptr, nullptr, nullptr, 0,
                  glogits, glogp, rows_per_g, g_scale, gentropy, gtop, top_ids, (int)top_k};
  if (short_rows(sa, dtype, (hipStream_t)stream, &rc)) return rc;
  GradArgs a = {};
  a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
  a.scale2 = kLog2e; a.inv_tau = 1.0f; a.stats_in = stats;
  a.tokens = tokens; a.token_bytes = token_bytes; a.entropy = entropy; a.glogp = glogp; a.rows_per_g = rows_per_g;
  a.g_scale = g_scale; a.gentropy = gentropy; a.gtop = top_k ? gtop : nullptr; a.top_ids = top_ids; a.top_k = (int)top_k;
  VAE_BY_TYPE(dtype, return (bwd_type<T, false>(a, (hipStream_t)stream)));
  return VAE_ERR_ARG;
}

int vae_token_nll_fused(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp,
                        float* stats, void* glogits, float grad_scale, void* scratch, int64_t N, int64_t V, int dtype,
                        vae_stream_t stream) {
  if (bad_rows(N, V, row_stride, dtype)) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !tokens || !logp || !stats || !glogits || (token_bytes != 4 && token_bytes != 8)) return VAE_ERR_ARG;
  int rc = VAE_ERR_ARG;
  ShortArgs sa = {logits, row_stride, tokens, token_bytes, N, (int)V, logp, nullptr, stats, nullptr, nullptr, 0,
                  glogits, nullptr, 1, -grad_scale, nullptr, nullptr, nullptr, 0};
  if (short_rows(sa, dtype, (hipStream_t)stream, &rc)) return rc;
  GradArgs a = {};
  a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
  a.scale2 = kLog2e; a.inv_tau = 1.0f;
  a.tokens = tokens; a.token_bytes = token_bytes; a.g_scale = grad_scale; a.out = logp; a.stats_out = stats;
  VAE_BY_TYPE(dtype, if (fused_type<T, false>(a, (hipStream_t)stream, &rc)) return rc);
  rc = vae_token_logp_fwd(logits, row_stride, tokens, token_bytes, logp, nullptr, stats, nullptr, nullptr, 0, scratch, N,
                          V, dtype, stream);
  if (rc != VAE_OK) return rc;
  return vae_token_logp_bwd(logits, row_stride, tokens, token_bytes, stats, nullptr, nullptr, 1, -grad_scale, nullptr,
                            nullptr, nullptr, 0, glogits, N, V, dtype, stream);
}

int vae_distill_bwd(const void* logits, int64_t row_stride, const void* t_logits, int64_t t_stride, int t_dtype,
                    const void* t_ids, int64_t id_stride, int id_bytes, int64_t K, float temperature,
                    const float* stats, const float* gkl, const float* gmean, float mean_scale, void* glogits,
                    int64_t N, int64_t V, int dtype, vae_stream_t stream) {
  if (K > VAE_MAX_TEACHER) return VAE_ERR_ARG;
  GradArgs a = {};
  a.teacher = {t_logits, t_ids, t_stride, id_stride, t_dtype, id_bytes, (int)K};
  if (bad_rows(N, V, row_stride, dtype) || bad_teacher(a.teacher, N, temperature)) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !t_logits || !t_ids || !stats || !glogits) return VAE_ERR_ARG;
  a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
  a.stats_in = stats; a.gkl = gkl; a.gmean = gmean; a.mean_scale = mean_scale;
  set_temperature(a, temperature);
  VAE_BY_TYPE(dtype, return (bwd_type<T, true>(a, (hipStream_t)stream)));
  return VAE_ERR_ARG;
}

int vae_distill_fwd(const void* logits, int64_t row_stride, const void* t_logits, int64_t t_stride, int t_dtype,
                    const void* t_ids, int64_t id_stride, int id_bytes, int64_t K, float temperature, float* kl,
                    float* stats, void* glogits, float grad_scale, void* scratch, int64_t N, int64_t V, int dtype,
                    vae_stream_t stream) {
  if (K > VAE_MAX_TEACHER) return VAE_ERR_ARG;
  GradArgs a = {};
  a.teacher = {t_logits, t_ids, t_stride, id_stride, t_dtype, id_bytes, (int)K};
  if (bad_rows(N, V, row_stride, dtype) || bad_teacher(a.teacher, N, temperature)) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !t_logits || !t_ids || !kl || (glogits && !stats)) return VAE_ERR_ARG;
  if (glogits) {
    a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
    a.mean_scale = grad_scale; a.out = kl; a.stats_out = stats;
    set_temperature(a, temperature);
    int rc = VAE_ERR_ARG;
    VAE_BY_TYPE(dtype, if (fused_type<T, true>(a, (hipStream_t)stream, &rc)) return rc);
  }
  const int rc = distill_stats(logits, row_stride, a.teacher, temperature, kl, stats, scratch, N, V, dtype,
                               (hipStream_t)stream);
  if (rc != VAE_OK || !glogits) return rc;
  return vae_distill_bwd(logits, row_stride, t_logits, t_stride, t_dtype, t_ids, id_stride, id_bytes, K, temperature,
                         stats, nullptr, nullptr, grad_scale, glogits, N, V, dtype, stream);
}

}  // extern "C"
