// Forward over rows of logits [N, V]: log probabilities of given tokens, entropy, top alternatives, and the KL from a
// teacher's top logits.  Formulas and the conventions for masks: token_row.hpp.
//   log p_t,   H = ln2 (log2 s - sum d 2^d / s) with d = (x - m) log2(e),   top k by (value, lower index first)
//   KL = sum_k q_k (ln q_k - ln p_id_k),  q the teacher's softmax over its entries
// A row whose token is negative is padding: none of its logits is read.
//
// One pass over the logits: every thread keeps a running (max, sum, weighted sum) of its vectors, merged across the
// workgroup at the end, so a row is read once whatever its length.  Few rows are cut into `parts` pieces of one
// workgroup each, whose partial results a second launch joins.
#include "token_row.hpp"

namespace vae {

constexpr int kCand = 1024;          // candidates for the alternatives that LDS holds
constexpr int kVecBytes = 16;
constexpr float kHuge = 1.0e6f;      // |max| beyond which the shifted exponent is formed as (x - m) c, see row_stats

struct FwdArgs {
  const void* logits;
  int64_t row_stride;
  const void* tokens;
  int token_bytes;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_ids;
  int top_k;
  int64_t N;
  int V;
  int parts, part_vecs;              // pieces of a row, vectors per piece
  char* scratch;                     // per (row, piece): m, s, t, -, then top_k keys
  float scale2, inv_tau;
  TeacherArgs teacher;
};
__device__ __forceinline__ int64_t part_bytes(int top_k) { return 16 + 8 * (int64_t)top_k; }

// One thread's running statistics.  With the reference r = max(m, -kHuge) and S = r c rounded once, e_j = 2^(x_j c - S)
// takes one fma and one exponential an element; S is the same for the whole sum, so its rounding drops out (finish()).
template <bool ENT>
struct RunStats {
  float m = -INFINITY, S, s = 0.f, t = 0.f;
  __device__ __forceinline__ explicit RunStats(float c) : S(mul_rn(-kHuge, c)) {}
  // make room for a maximum of mt
  __device__ __forceinline__ void raise(float mt, float c) {
    m = max_raw(m, mt);
    const float Sn = mul_rn(max_raw(m, -kHuge), c);   // rounded here, not fused into the difference below
    const float w = exp2_raw(S - Sn);
    if constexpr (ENT) t = w * __builtin_fmaf(S - Sn, s, t);
    s *= w;
    S = Sn;
  }
  __device__ __forceinline__ void add(float x, float c) {
    const float d = __builtin_fmaf(x, c, -S);
    const float e = exp2_raw(d);
    s += e;
    if constexpr (ENT) t = __builtin_fmaf(max_raw(d, -300.f), e, t);  // -inf times 0 would be NaN
  }
};

// Statistics of vectors [v0, v1) of a row (and its edges when they belong to this piece), for the whole workgroup.
// On return m, s, t are the workgroup's, relative to the exact maximum; `tile` is the thread's first vector group that
// reached its own maximum `mine` (for the alternatives), -1 if it has none.
template <typename T, int BT, bool ENT>
__device__ __forceinline__ void row_stats(const T* __restrict__ x, const RowCut<T, VecOf<T>::n>& cut, int v0, int v1,
                                          float edge, bool has_edge, float c, float& m, float& s, float& t, float& mine,
                                          int& tile) {
  constexpr int VN = VecOf<T>::n, U = 4;
  const Buffer body(x + cut.head, cut.nvec * kVecBytes);
  RunStats<ENT> st(c);
  tile = -1;
  int j = v0 + (int)threadIdx.x;
  const int full = (v1 - v0) / (U * BT);
  if (j < v1) tile = j;
  for (int it = 0; it < full; ++it, j += U * BT) {
    Packet<T, VN> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p[u].load(body, j * kVecBytes, u * BT * kVecBytes);
    float v[U][VN], mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u].get(v[u]);
      mt = vec_max(v[u], mt);
    }
    if (mt > st.m) tile = j;
    st.raise(mt, c);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VN; ++i) st.add(v[u][i], c);
  }
  for (; j < v1; j += BT) {
    Packet<T, VN> p;
    p.load(body, j * kVecBytes, 0);
    float v[VN];
    p.get(v);
    const float mt = vec_max(v, -INFINITY);
    if (mt > st.m) tile = j;
    st.raise(mt, c);
#pragma unroll
    for (int i = 0; i < VN; ++i) st.add(v[i], c);
  }
  mine = st.m;
  if (has_edge) {
    st.raise(edge, c);
    st.add(edge, c);
  }
  m = block_max<BT>(st.m);
  if (!(fabsf(m) > kHuge) || m == -INFINITY) {
    st.raise(m, c);
    s = block_sum<BT>(st.s);
    if constexpr (ENT) t = block_sum<BT>(st.t);
    // relative to the exact maximum: 2^(x c - S) = 2^((x - m) c) 2^(m c - S)
    const float r = m == -INFINITY ? 0.f : __builtin_fmaf(m, c, -st.S);
    const float w = exp2_raw(-r);
    if constexpr (ENT) t = w * __builtin_fmaf(-r, s, t);
    s *= w;
    return;
  }
  // a maximum so large that x c - S loses it: once more, the difference first
  s = t = 0.f;
  auto add = [&](float v) {
    const float d = (v - m) * c;
    const float e = exp2_raw(d);
    s += e;
    if constexpr (ENT) t = __builtin_fmaf(max_raw(d, -300.f), e, t);
  };
  for (j = v0 + (int)threadIdx.x; j < v1; j += BT) {
    Packet<T, VN> p;
    p.load(body, j * kVecBytes, 0);
    float v[VN];
    p.get(v);
#pragma unroll
    for (int i = 0; i < VN; ++i) add(v[i]);
  }
  if (has_edge) add(edge);
  s = block_sum<BT>(s);
  if constexpr (ENT) t = block_sum<BT>(t);
}

// ---------------------------------------------------------------------------------------------------------------
// The k largest keys of a set.  Every thread brings the largest key of its own share; the k-th largest of those is a
// lower bound of the k-th largest of all, and only the k threads at or above it can hold any of the k.
// ---------------------------------------------------------------------------------------------------------------
template <int BT>
struct TopLds {
  uint64_t keys[BT], cand[kCand];
  int seg[BT];
  int nseg, ncand;
  uint64_t bound;
};

// the k-th largest of the BT keys in lds.keys (0 where fewer than k are there): bit by bit, by the first wave
template <int BT>
__device__ __forceinline__ uint64_t kth_key(TopLds<BT>& lds, uint64_t mine, int k) {
  lds_barrier();
  lds.keys[threadIdx.x] = mine;
  if (threadIdx.x == 0) lds.nseg = lds.ncand = 0;
  lds_barrier();
  if (threadIdx.x < 64) {
    uint64_t key[BT / 64];
#pragma unroll
    for (int i = 0; i < BT / 64; ++i) key[i] = lds.keys[threadIdx.x + 64 * i];
    uint64_t b = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t want = b | (1ull << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < BT / 64; ++i) n += __popcll(__ballot(key[i] >= want));
      if (n >= k) {
        b = want;
        if (n == k) break;
      }
    }
    if (threadIdx.x == 0) lds.bound = b;
  }
  lds_barrier();
  return lds.bound;
}

template <int BT>
__device__ __forceinline__ void push_key(TopLds<BT>& lds, uint64_t key, uint64_t bound) {
  if (key != 0 && key >= bound) {
    const int at = atomicAdd(&lds.ncand, 1);
    if (at < kCand) lds.cand[at] = key;
  }
}

// emit(rank, key) for the candidates of rank < k; key 0 for the ranks that are not there.  False: too many candidates.
template <int BT, typename Emit>
__device__ __forceinline__ bool emit_ranked(TopLds<BT>& lds, int k, Emit emit) {
  lds_barrier();
  const int n = lds.ncand;
  if (n > kCand) return false;
  for (int i = threadIdx.x; i < n; i += BT) {
    const uint64_t key = lds.cand[i];
    int rank = 0;
    for (int q = 0; q < n; ++q) rank += lds.cand[q] > key ? 1 : 0;
    if (rank < k) emit(rank, key);
  }
  for (int i = n + threadIdx.x; i < k; i += BT) emit(i, (uint64_t)0);
  return true;
}

// The k largest of vectors [v0, v1) and the edges of a row; `mine`, `tile` from row_stats.
template <typename T, int BT, typename Emit>
__device__ __forceinline__ void row_top(TopLds<BT>& lds, const T* __restrict__ x, const RowCut<T, VecOf<T>::n>& cut,
                                        int v0, int v1, float edge, int edge_index, float mine, int tile, int k,
                                        Emit emit) {
  constexpr int VN = VecOf<T>::n, U = 4;
  const Buffer body(x + cut.head, cut.nvec * kVecBytes);
  auto vec_key = [&](int j, int i, float v) { return order_key(v, (uint32_t)(cut.index(j) + i)); };
  uint64_t key = edge_index >= 0 ? order_key(edge, (uint32_t)edge_index) : 0;
  if (tile >= 0) {
    // the first element of the thread's share that is its maximum: somewhere in `tile`
    uint64_t best = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = tile + u * BT;
      if (j < v1) {
        Packet<T, VN> p;
        p.load(body, j * kVecBytes, 0);
        float v[VN];
        p.get(v);
#pragma unroll
        for (int i = 0; i < VN; ++i)
          if (v[i] == mine && best == 0) best = vec_key(j, i, v[i]);
      }
    }
    key = best > key ? best : key;
  }
  const uint64_t bound = kth_key(lds, key, k);
  if (key != 0 && key >= bound) lds.seg[atomicAdd(&lds.nseg, 1)] = threadIdx.x;
  if (edge_index >= 0) push_key(lds, order_key(edge, (uint32_t)edge_index), bound);
  lds_barrier();
  const int nseg = lds.nseg, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int q = wave; q < nseg; q += BT / 64) {
    for (int j = v0 + lds.seg[q] + lane * BT; j < v1; j += 64 * BT) {
      Packet<T, VN> p;
      p.load(body, j * kVecBytes, 0);
      float v[VN];
      p.get(v);
#pragma unroll
      for (int i = 0; i < VN; ++i) push_key(lds, vec_key(j, i, v[i]), bound);
    }
  }
  if (emit_ranked(lds, k, emit)) return;
  // the large values all sit in few threads' shares: one after the other
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = edge_index >= 0 ? order_key(edge, (uint32_t)edge_index) : 0;
    if (best >= last) best = 0;
    for (int j = v0 + (int)threadIdx.x; j < v1; j += BT) {
      Packet<T, VN> p;
      p.load(body, j * kVecBytes, 0);
      float v[VN];
      p.get(v);
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const uint64_t kk = vec_key(j, i, v[i]);
        if (kk < last && kk > best) best = kk;
      }
    }
    last = block_max_key<BT>(best);
    if (threadIdx.x == 0) emit(r, last);
  }
}

__device__ __forceinline__ void emit_top(const FwdArgs& a, int64_t row, int rank, uint64_t key, float m, float s) {
  a.top_logp[row * a.top_k + rank] = key ? row_log_prob(key_value(key), m, s, 1.0f) : nan_f();
  a.top_ids[row * a.top_k + rank] = key ? key_index(key) : -1;
}
template <int BT>
__device__ __forceinline__ void write_padding(const FwdArgs& a, int64_t row) {
  if (threadIdx.x == 0) {
    if (a.logp) a.logp[row] = 0.f;
    if (a.entropy) a.entropy[row] = 0.f;
    if (a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.f;
  }
  for (int i = threadIdx.x; i < a.top_k; i += BT) {
    a.top_logp[row * a.top_k + i] = -INFINITY;
    a.top_ids[row * a.top_k + i] = -1;
  }
}
// what a row's statistics give, once they are whole
template <typename T, int BT, bool ENT, bool DIST>
__device__ __forceinline__ void write_row(const FwdArgs& a, int64_t row, const T* __restrict__ x, int64_t tok, float m,
                                          float s, float t, const TeacherRow<BT>* tr) {
  float kl = 0.f;
  if constexpr (DIST) {
    for (int k = threadIdx.x; k < a.teacher.K; k += BT)
      if (tr->id[k] >= 0) kl += tr->q[k] * (tr->logq[k] - row_log_prob(to_f32(x[tr->id[k]]), m, s, a.inv_tau));
    kl = block_sum<BT>(kl);
  }
  if (threadIdx.x == 0) {
    if constexpr (DIST) a.logp[row] = kl;
    else if (a.logp) a.logp[row] = tok < a.V ? row_log_prob(to_f32(x[tok]), m, s, 1.0f) : nan_f();
    if constexpr (ENT) a.entropy[row] = s == 0.f ? 0.f : kLn2 * (log2f(s) - t / s);
    if (a.stats) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = s;
    }
  }
}

template <typename T, int BT, bool ENT, bool TOP, bool DIST>
__global__ __launch_bounds__(BT) void token_fwd_kernel(FwdArgs a) {
  constexpr int VN = VecOf<T>::n;
  __shared__ struct {
    TopLds<TOP ? BT : 64> top[TOP ? 1 : 0];
    TeacherRow<BT> teacher[DIST ? 1 : 0];
  } lds;
  for (int64_t item = blockIdx.x; item < a.N * a.parts; item += gridDim.x) {
    const int64_t row = a.parts == 1 ? item : item / a.parts;
    const int part = a.parts == 1 ? 0 : (int)(item - row * a.parts);
    const T* x = (const T*)a.logits + row * a.row_stride;
    int64_t tok = 0;
    if constexpr (DIST) {
      if (a.parts == 1) {
        const int state = lds.teacher[0].load(a.teacher, row, a.V, a.inv_tau, a.scale2);
        if (state != kRowFine) {
          if (threadIdx.x == 0) {
            a.logp[row] = state == kRowEmpty ? 0.f : nan_f();
            if (a.stats) a.stats[2 * row] = 0.f, a.stats[2 * row + 1] = a.logp[row];  // the backward's sign of either
          }
          continue;
        }
      }
    } else {
      tok = a.tokens ? load_id(a.tokens, a.token_bytes, row) : 0;
      if (tok < 0) {
        if (a.parts == 1) write_padding<BT>(a, row);
        continue;
      }
    }
    const RowCut<T, VN> cut(x, a.V);
    const int v0 = part * a.part_vecs;
    int v1 = v0 + a.part_vecs;
    v1 = v1 < cut.nvec ? v1 : cut.nvec;
    int ei = cut.edge(threadIdx.x);
    if (ei >= 0 && (ei < cut.head ? part != 0 : part != a.parts - 1)) ei = -1;  // the head goes with the first piece
    const float edge = ei >= 0 ? to_f32(x[ei]) : -INFINITY;
    float m, s, t = 0.f, mine;
    int tile;
    row_stats<T, BT, ENT>(x, cut, v0, v1, edge, ei >= 0, a.scale2, m, s, t, mine, tile);
    if (a.parts == 1) {
      if constexpr (TOP)
        row_top<T, BT>(lds.top[0], x, cut, v0, v1, edge, ei, mine, tile, a.top_k,
                       [&](int rank, uint64_t key) { emit_top(a, row, rank, key, m, s); });
      write_row<T, BT, ENT, DIST>(a, row, x, tok, m, s, t, lds.teacher);
    } else {
      char* to = a.scratch + item * part_bytes(a.top_k);
      if (threadIdx.x == 0) {
        float* f = reinterpret_cast<float*>(to);
        f[0] = m;
        f[1] = s;
        f[2] = t;
      }
      if constexpr (TOP)
        row_top<T, BT>(lds.top[0], x, cut, v0, v1, edge, ei, mine, tile, a.top_k,
                       [&](int rank, uint64_t key) { reinterpret_cast<uint64_t*>(to + 16)[rank] = key; });
    }
  }
}

// joins the pieces of a row: one workgroup a row
template <typename T, int BT, bool ENT, bool TOP, bool DIST>
__global__ __launch_bounds__(BT) void token_join_kernel(FwdArgs a) {
  __shared__ struct {
    TopLds<TOP ? BT : 64> top[TOP ? 1 : 0];
    TeacherRow<BT> teacher[DIST ? 1 : 0];
  } lds;
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* x = (const T*)a.logits + row * a.row_stride;
    int64_t tok = 0;
    if constexpr (DIST) {
      const int state = lds.teacher[0].load(a.teacher, row, a.V, a.inv_tau, a.scale2);
      if (state != kRowFine) {
        if (threadIdx.x == 0) {
          a.logp[row] = state == kRowEmpty ? 0.f : nan_f();
          if (a.stats) a.stats[2 * row] = 0.f, a.stats[2 * row + 1] = a.logp[row];
        }
        continue;
      }
    } else {
      tok = a.tokens ? load_id(a.tokens, a.token_bytes, row) : 0;
      if (tok < 0) {
        write_padding<BT>(a, row);
        continue;
      }
    }
    const char* from = a.scratch + row * a.parts * part_bytes(a.top_k);
    float mp = -INFINITY, sp = 0.f, tp = 0.f;
    if ((int)threadIdx.x < a.parts) {   // parts <= BT
      const float* f = reinterpret_cast<const float*>(from + threadIdx.x * part_bytes(a.top_k));
      mp = f[0];
      sp = f[1];
      tp = f[2];
    }
    const float m = block_max<BT>(mp);
    const float d = sp == 0.f ? 0.f : (mp - m) * a.scale2;
    const float w = exp2_raw(d);
    const float s = block_sum<BT>(w * sp);
    float t = 0.f;
    if constexpr (ENT) t = block_sum<BT>(w * __builtin_fmaf(max_raw(d, -300.f), sp, tp));
    if constexpr (TOP) {
      const int n = a.parts * a.top_k;
      auto key_at = [&](int i) {
        const int p = i / a.top_k;
        return reinterpret_cast<const uint64_t*>(from + p * part_bytes(a.top_k) + 16)[i - p * a.top_k];
      };
      auto emit = [&](int rank, uint64_t key) { emit_top(a, row, rank, key, m, s); };
      uint64_t mine = 0;
      for (int i = threadIdx.x; i < n; i += BT) {
        const uint64_t key = key_at(i);
        mine = key > mine ? key : mine;
      }
      const uint64_t bound = kth_key(lds.top[0], mine, a.top_k);
      for (int i = threadIdx.x; i < n; i += BT) push_key(lds.top[0], key_at(i), bound);
      if (!emit_ranked(lds.top[0], a.top_k, emit)) {
        uint64_t last = ~0ull;
        for (int r = 0; r < a.top_k; ++r) {
          uint64_t best = 0;
          for (int i = threadIdx.x; i < n; i += BT) {
            const uint64_t key = key_at(i);
            if (key < last && key > best) best = key;
          }
          last = block_max_key<BT>(best);
          if (threadIdx.x == 0) emit(r, last);
        }
      }
    }
    write_row<T, BT, ENT, DIST>(a, row, x, tok, m, s, t, lds.teacher);
  }
}

static bool bad_shape(int64_t N, int64_t V, int64_t row_stride, int dtype) {
  return N < 0 || V < 1 || V > VAE_MAX_ROW || (N > 1 && row_stride < V) ||
         (dtype != VAE_F32 && dtype != VAE_BF16 && dtype != VAE_F16);
}
static int grid_for(int64_t items) { return (int)(items < kMaxGrid ? items : kMaxGrid); }

// Pieces of a row: with fewer than kFillRows rows a workgroup a row leaves compute units idle; a piece keeps at least
// kPieceVecs vectors, so that the join's cost stays below what the split saves.
constexpr int64_t kFillRows = 512, kPieceVecs = 512;
struct Cut {
  int parts, part_vecs;
};
static Cut cut_rows(int64_t N, int64_t V, int dtype) {
  const int64_t vn = dtype == VAE_F32 ? 4 : 8;
  const int64_t nvec = (V + vn - 1) / vn;
  int64_t parts = 1;
  if (N < kFillRows) {
    parts = 2 * kFillRows / (N > 0 ? N : 1);
    const int64_t most = nvec / kPieceVecs;
    parts = parts < most ? parts : most;
    parts = parts < 1 ? 1 : (parts > kBlock ? kBlock : parts);
  }
  const int64_t per = (nvec + parts - 1) / parts;
  return {(int)((nvec + per - 1) / per), (int)per};
}
// rows of up to this many vectors take one wave each
constexpr int64_t kWaveVecs = 512;

template <typename T, int BT, bool ENT, bool TOP, bool DIST>
static int fwd_launch(const FwdArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((token_fwd_kernel<T, BT, ENT, TOP, DIST>), dim3(grid_for(a.N * a.parts)), dim3(BT), 0, st, a);
  if (a.parts > 1)
    hipLaunchKernelGGL((token_join_kernel<T, kBlock, ENT, TOP, DIST>), dim3(grid_for(a.N)), dim3(kBlock), 0, st, a);
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
}
template <typename T, bool DIST>
static int fwd_type(const FwdArgs& a, hipStream_t st) {
  const bool wave = a.parts == 1 && (a.V + VecOf<T>::n - 1) / VecOf<T>::n <= kWaveVecs;
#define VAE_FWD(E, K) (wave ? fwd_launch<T, 64, E, K, DIST>(a, st) : fwd_launch<T, kBlock, E, K, DIST>(a, st))
  if constexpr (DIST) return VAE_FWD(false, false);
  else {
    if (a.entropy) return a.top_k ? VAE_FWD(true, true) : VAE_FWD(true, false);
    return a.top_k ? VAE_FWD(false, true) : VAE_FWD(false, false);
  }
#undef VAE_FWD
}

// kl and stats; vae_distill_fwd (token_grad.hip) has checked the arguments
int distill_stats(const void* logits, int64_t row_stride, const TeacherArgs& teacher, float temperature, float* kl,
                  float* stats, void* scratch, int64_t N, int64_t V, int dtype, hipStream_t stream) {
  const Cut cut = cut_rows(N, V, dtype);
  if (cut.parts > 1 && !scratch) return VAE_ERR_ARG;
  const FwdArgs a = {logits, row_stride, nullptr, 0, kl, nullptr, stats, nullptr, nullptr, 0, N, (int)V, cut.parts,
                     cut.part_vecs, (char*)scratch, (float)(1.4426950408889634 / (double)temperature),
                     (float)(1.0 / (double)temperature), teacher};
  VAE_BY_TYPE(dtype, return (fwd_type<T, true>(a, stream)));
  return VAE_ERR_ARG;
}

}  // namespace vae

using namespace vae;

extern "C" {

size_t vae_token_scratch_bytes(int64_t N, int64_t V, int64_t top_k, int dtype) {
  if (N < 1 || V < 1 || V > VAE_MAX_ROW || top_k < 0 || top_k > VAE_MAX_TOP) return 0;
  const Cut c = cut_rows(N, V, dtype);
  return c.parts == 1 ? 0 : (size_t)N * c.parts * (16 + 8 * (size_t)top_k);
}

int vae_token_logp_fwd(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp,
                       float* entropy, float* stats, float* top_logp, int64_t* top_ids, int64_t top_k, void* scratch,
                       int64_t N, int64_t V, int dtype, vae_stream_t stream) {
  if (bad_shape(N, V, row_stride, dtype) || top_k < 0 || top_k > VAE_MAX_TOP || top_k > V) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || (tokens && token_bytes != 4 && token_bytes != 8)) return VAE_ERR_ARG;
  if ((logp && !tokens) || (top_k > 0 && (!top_logp || !top_ids))) return VAE_ERR_ARG;
  int rc = VAE_OK;
  ShortArgs sa = {logits, row_stride, tokens, token_bytes, N, (int)V, logp, entropy, stats, top_logp, top_ids, (int)top_k};
  if (short_rows(sa, dtype, (hipStream_t)stream, &rc)) return rc;
  const Cut cut = cut_rows(N, V, dtype);
  if (cut.parts > 1 && !scratch) return VAE_ERR_ARG;
  const FwdArgs a = {logits, row_stride, tokens, token_bytes, logp, entropy, stats, top_logp, top_ids, (int)top_k, N,
                     (int)V, cut.parts, cut.part_vecs, (char*)scratch, kLog2e, 1.0f, {}};
  VAE_BY_TYPE(dtype, return (fwd_type<T, false>(a, (hipStream_t)stream)));
  return VAE_ERR_ARG;
}

}  // extern "C"
