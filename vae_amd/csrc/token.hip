// Forward over rows of logits [N, V]: log probabilities of given tokens, entropy, top alternatives, and the KL from a
// teacher's top logits.  Formulas and the conventions for masks: token_row.hpp.
//   log p_t,   H = ln2 (log2 s - sum d 2^d / s) with d = (x - m) log2(e),   top k by (value, lower index first)
//   KL = sum_k q_k (ln q_k - ln p_id_k),  q the teacher's softmax over its entries
// A row whose token is negative is padding: none of its logits is read.
//
// One pass over the logits: every thread keeps a running (max, sum, weighted sum) of its vectors, merged across the
// workgroup at the end, so a row is read once whatever its length.  Few rows are cut into `parts` pieces of one
// workgroup each, whose partial results a second launch joins.  Bound by the read: 4096 x 32768 bf16 with entropy 44 us
// (6.1 TB/s), 2048 x 50021 fp16 (rows at every alignment) 39 us (5.3 TB/s); the arithmetic is an fma, an exponential and
// an addition an element, two more with the entropy.
#include "token_row.hpp"

namespace vae {

constexpr int kVecBytes = 16;
constexpr float kHuge = 1.0e6f;      // |max c| beyond which the shifted exponent is formed as (x - m) c, see row_stats

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
  Teacher teacher;
};
__device__ __forceinline__ int64_t part_bytes(int top_k) { return 16 + 8 * (int64_t)top_k; }

// One thread's running statistics.  With the reference S = max(m c, -kHuge) rounded once, e_j = 2^(x_j c - S) takes one
// fma and one exponential an element; S is the same for the whole sum, so its rounding drops out at the end of row_stats,
// which takes these sums where |max c| <= kHuge: S is at most 2^-5 off there.  Beyond it (large logits, a small temperature)
// the rounding of S alone could carry a sum out of the type's range.
template <bool ENT>
struct RunStats {
  float m = -INFINITY, S = -kHuge, s = 0.f, t = 0.f;
  // make room for a maximum of mt
  __device__ __forceinline__ void raise(float mt, float c) {
    m = max_raw(m, mt);
    const float Sn = max_raw(mul_rn(m, c), -kHuge);   // rounded here, not fused into the difference below
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
// On return m, s, t are the workgroup's, relative to the exact maximum; `mine` is the thread's own maximum (without the
// edge), for the alternatives.  NT: the row is not read again.
template <typename T, int BT, bool ENT, bool NT>
__device__ __forceinline__ void row_stats(const T* __restrict__ x, const RowCut<T, VecOf<T>::n>& cut, int v0, int v1,
                                          float edge, bool has_edge, float c, float& m, float& s, float& t,
                                          float& mine) {
  constexpr int VN = VecOf<T>::n, U = 4;
  const Buffer body(x + cut.head, cut.nvec * kVecBytes);
  RunStats<ENT> st;
  // W vectors of a lane; a running maximum for all of them
  auto group = [&](auto& p) {
    constexpr int W = sizeof(p) / sizeof(p[0]);
    float v[W][VN], mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      p[u].get(v[u]);
      mt = vec_max(v[u], mt);
    }
    st.raise(mt, c);
#pragma unroll
    for (int u = 0; u < W; ++u) {
#pragma unroll
      for (int i = 0; i < VN; ++i) st.add(v[u][i], c);
      __builtin_amdgcn_sched_barrier(0);   // vector by vector: interleaved they need half as many registers again
    }
  };
  int j = v0 + (int)threadIdx.x;
  const int full = (v1 - v0) / (U * BT);
  for (int it = 0; it < full; ++it, j += U * BT) {
    Packet<T, VN> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p[u].template load<NT>(body, j * kVecBytes, u * BT * kVecBytes);
    group(p);
  }
  for (; j < v1; j += BT) {
    Packet<T, VN> p[1];
    p[0].template load<NT>(body, j * kVecBytes);
    group(p);
  }
  mine = st.m;
  if (has_edge) {
    st.raise(edge, c);
    st.add(edge, c);
  }
  m = block_max<BT>(st.m);
  if (!(fabsf(m) * c > kHuge) || m == -INFINITY) {
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
  // a maximum so large that x c - S loses the difference: once more, the difference first
  s = t = 0.f;
  auto add = [&](float v) {
    const float d = (v - m) * c;
    const float e = exp2_raw(d);
    s += e;
    if constexpr (ENT) t = __builtin_fmaf(max_raw(d, -300.f), e, t);
  };
  for (j = v0 + (int)threadIdx.x; j < v1; j += BT) {
    Packet<T, VN> p;
    p.template load<NT>(body, j * kVecBytes);
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
// The k largest keys (order_key: value, then the lower index) of what a workgroup has read.  A bound from below comes
// from the threads' own maxima: every wave takes the ceil(k / waves)-th largest of its lanes', the least of those has k
// elements at or above it.  Only the few threads whose maximum reaches the bound can hold any of the k; their vectors
// are read once more (out of the caches), all lanes side by side.  4096 x 32768 bf16, k = 20: 67 us, 57 for k = 4, 44
// without alternatives; a list kept while reading costs every element a comparison (145 us).
// ---------------------------------------------------------------------------------------------------------------
constexpr int kCand = 1024;      // candidates that LDS holds
constexpr int kMostShares = 96;  // threads at the bound beyond which equal values are told apart by their index first

template <int BT>
struct TopLds {
  uint64_t cand[kCand];
  uint64_t wave_bound[BT / 64];
  int share[BT];
  int nshare, ncand;
};

// the n-th largest of a wave's 64 keys, its bits below `last` cleared; 0 where there are fewer than n
__device__ __forceinline__ uint64_t wave_nth(uint64_t key, int n, int last) {
  uint64_t b = 0;
  for (int bit = 63; bit >= last; --bit) {
    const uint64_t want = b | (1ull << bit);
    b = __popcll(__ballot(key >= want)) >= n ? want : b;
  }
  return b;
}
// the least of the first `waves` waves' `each`-th largest keys: waves * each keys are at or above it
template <int BT>
__device__ __forceinline__ uint64_t block_bound(TopLds<BT>& lds, uint64_t key, int each, int waves, int last) {
  const uint64_t mine = wave_nth(key, each, last);
  lds_barrier();   // what the last one left has been read
  if ((threadIdx.x & 63) == 0) lds.wave_bound[threadIdx.x >> 6] = mine;
  if (threadIdx.x == 0) lds.nshare = lds.ncand = 0;
  lds_barrier();
  uint64_t b = lds.wave_bound[0];
  for (int w = 1; w < waves; ++w) b = lds.wave_bound[w] < b ? lds.wave_bound[w] : b;
  return b;
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
#pragma unroll 4
    for (int q = 0; q < n; ++q) rank += lds.cand[q] > key ? 1 : 0;
    if (rank < k) emit(rank, key);
  }
  for (int i = n + threadIdx.x; i < k; i += BT) emit(i, (uint64_t)0);
  return true;
}

template <typename T, int BT, typename Emit>
__device__ __forceinline__ void row_top(TopLds<BT>& lds, const T* __restrict__ x, const RowCut<T, VecOf<T>::n>& cut,
                                        int v0, int v1, float edge, int edge_index, float mine, int k, Emit emit) {
  constexpr int VN = VecOf<T>::n;
  // How far the bound is worked out: sign, exponent and 7 bits of the fraction tell two bf16 numbers apart; fp16 (10 bits)
  // and fp32 may find a bound a little lower and with it a few more candidates
  constexpr int kLastBit = sizeof(T) == 2 ? 48 : 40;
  const Buffer body(x + cut.head, cut.nvec * kVecBytes);
  const int tid = threadIdx.x;
  auto each = [&](int j, auto f) {   // the elements of vector j
    Packet<T, VN> p;
    p.template load<false>(body, j * kVecBytes);
    float v[VN];
    p.get(v);
#pragma unroll
    for (int i = 0; i < VN; ++i) f(v[i], (uint32_t)(cut.index(j) + i));
  };
  const uint64_t edge_key = edge_index >= 0 ? order_key(edge, (uint32_t)edge_index) : 0;
  uint64_t key = v0 + tid < v1 ? (uint64_t)order_bits(mine) << 32 : 0;
  const uint64_t edge_top = edge_key >> 32 << 32;
  key = edge_top > key ? edge_top : key;
  constexpr int NW = BT / 64;
  uint64_t bound = block_bound(lds, key, (k + NW - 1) / NW, NW, kLastBit);
  auto take_share = [&]() {
    if (key != 0 && key >= bound) lds.share[atomicAdd(&lds.nshare, 1)] = tid;
    lds_barrier();
    return lds.nshare;
  };
  int n = take_share();
  if (n > kMostShares) {
    // many equal maxima (a constant row, a mask that leaves little): the first index of each decides
    key = edge_key;
    uint64_t best = 0;
    for (int j = v0 + tid; j < v1 && best == 0; j += BT)
      each(j, [&](float v, uint32_t at) { best = v == mine && best == 0 ? order_key(v, at) : best; });
    key = best > key ? best : key;
    bound = block_bound(lds, key, (k + NW - 1) / NW, NW, 0);
    n = take_share();
  }
  push_key(lds, edge_key, bound);
  // the shares' vectors, side by side: share q holds v0 + share[q] + i BT
  const int per = (v1 - v0 + BT - 1) / BT;
  const float least = (bound >> 32) > order_bits(-INFINITY) ? key_value(bound) : -INFINITY;   // below it lie the NaN
  for (int q = tid; q < n * per; q += BT) {
    const int j = v0 + lds.share[q / per] + (q % per) * BT;
    if (j < v1) {
      each(j, [&](float v, uint32_t at) {
        if (v >= least) push_key(lds, order_key(v, at), bound);
      });
    }
  }
  if (emit_ranked(lds, k, emit)) return;
  // the large values all sit in few threads' shares: one after the other
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = edge_key < last ? edge_key : 0;
    for (int j = v0 + tid; j < v1; j += BT)
      each(j, [&](float v, uint32_t at) {
        const uint64_t kk = order_key(v, at);
        best = kk < last && kk > best ? kk : best;
      });
    last = block_max_key<BT>(best);
    if (tid == 0) emit(r, last);
  }
}

__device__ __forceinline__ void emit_top(const FwdArgs& a, int64_t row, int rank, uint64_t key, float m, float s) {
  a.top_logp[row * a.top_k + rank] = key ? row_log_prob(key_value(key), m, s, 1.0f) : nan_f();
  a.top_ids[row * a.top_k + rank] = key ? key_index(key) : -1;
}
// true: the row is done, one without entries or with an id beyond the vocabulary
__device__ __forceinline__ bool write_no_teacher(const FwdArgs& a, int64_t row, bool write) {
  const int state = a.teacher.state[row];
  if (state != kRowFine && write && threadIdx.x == 0) {
    const float v = state == kRowEmpty ? 0.f : nan_f();
    a.logp[row] = v;
    if (a.stats) a.stats[2 * row] = 0.f, a.stats[2 * row + 1] = v;   // a sum of 0 or NaN: what the backward goes by
  }
  return state != kRowFine;
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
template <int BT, bool ENT, bool DIST>
__device__ __forceinline__ void write_row(const FwdArgs& a, int64_t row, int64_t tok, float token_logit, float m, float s,
                                          float t, const TeacherTerms<BT>& terms) {
  float kl = 0.f;
  if constexpr (DIST) kl = terms.kl(a.teacher.K, m, s, a.inv_tau);
  if (threadIdx.x == 0) {
    if constexpr (DIST) a.logp[row] = kl;
    else if (a.logp) a.logp[row] = tok < a.V ? row_log_prob(token_logit, m, s, 1.0f) : nan_f();
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
  } lds;
  for (int64_t item = blockIdx.x; item < a.N * a.parts; item += gridDim.x) {
    const int64_t row = a.parts == 1 ? item : item / a.parts;
    const int part = a.parts == 1 ? 0 : (int)(item - row * a.parts);
    const T* x = (const T*)a.logits + row * a.row_stride;
    int64_t tok = 0;
    float token_logit = 0.f;       // asked for in front of the row: it is there when the row's sum is
    TeacherTerms<BT> terms;
    if constexpr (DIST) {
      if (write_no_teacher(a, row, a.parts == 1)) continue;
      if (a.parts == 1) {
        terms.fetch(a.teacher, row);
        terms.fetch_logits(x);
      }
    } else {
      tok = a.tokens ? load_id(a.tokens, a.token_bytes, row) : 0;
      if (tok < 0) {
        if (a.parts == 1) write_padding<BT>(a, row);
        continue;
      }
      if (tok < a.V && a.parts == 1) token_logit = to_f32(x[tok]);
    }
    const RowCut<T, VN> cut(x, a.V);
    const int v0 = part * a.part_vecs;
    int v1 = v0 + a.part_vecs;
    v1 = v1 < cut.nvec ? v1 : cut.nvec;
    int ei = cut.edge(threadIdx.x);
    if (ei >= 0 && (ei < cut.head ? part != 0 : part != a.parts - 1)) ei = -1;  // the head goes with the first piece
    const float edge = ei >= 0 ? to_f32(x[ei]) : -INFINITY;
    float m, s, t = 0.f, mine;
    row_stats<T, BT, ENT, !TOP>(x, cut, v0, v1, edge, ei >= 0, a.scale2, m, s, t, mine);
    if constexpr (TOP) {
      char* to = a.scratch + item * part_bytes(a.top_k) + 16;
      row_top<T, BT>(lds.top[0], x, cut, v0, v1, edge, ei, mine, a.top_k, [&](int rank, uint64_t key) {
        if (a.parts == 1) emit_top(a, row, rank, key, m, s);
        else reinterpret_cast<uint64_t*>(to)[rank] = key;
      });
    }
    if (a.parts == 1) {
      write_row<BT, ENT, DIST>(a, row, tok, token_logit, m, s, t, terms);
    } else if (threadIdx.x == 0) {
      float* f = reinterpret_cast<float*>(a.scratch + item * part_bytes(a.top_k));
      f[0] = m;
      f[1] = s;
      f[2] = t;
    }
  }
}

// joins the pieces of a row: one workgroup a row
template <typename T, int BT, bool ENT, bool TOP, bool DIST>
__global__ __launch_bounds__(BT) void token_join_kernel(FwdArgs a) {
  __shared__ struct {
    TopLds<TOP ? BT : 64> top[TOP ? 1 : 0];
  } lds;
  constexpr int R = kCand / BT;     // keys a thread holds; more of them are read where they are
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* x = (const T*)a.logits + row * a.row_stride;
    // everything that does not depend on anything else is on its way first
    const char* from = a.scratch + row * a.parts * part_bytes(a.top_k);
    const int n = a.parts * a.top_k;
    const int at = (a.top_k + a.parts - 1) / a.parts - 1;   // a piece's keys are in order
    auto key_at = [&](int i) {
      const int p = i / a.top_k;
      return reinterpret_cast<const uint64_t*>(from + p * part_bytes(a.top_k) + 16)[i - p * a.top_k];
    };
    const int64_t tok = !DIST && a.tokens ? load_id(a.tokens, a.token_bytes, row) : 0;
    float mp = -INFINITY, sp = 0.f, tp = 0.f;
    if ((int)threadIdx.x < a.parts) {   // parts <= BT
      const float* f = reinterpret_cast<const float*>(from + threadIdx.x * part_bytes(a.top_k));
      mp = f[0];
      sp = f[1];
      tp = f[2];
    }
    uint64_t keys[TOP ? R : 1], lead = 0;
    if constexpr (TOP) {
#pragma unroll
      for (int r = 0; r < R; ++r) keys[r] = (int)threadIdx.x + r * BT < n ? key_at(threadIdx.x + r * BT) : 0;
      if ((int)threadIdx.x < a.parts) lead = key_at(threadIdx.x * a.top_k + at);
    }
    float token_logit = 0.f;
    TeacherTerms<BT> terms;
    if constexpr (DIST) {
      if (write_no_teacher(a, row, true)) continue;
      terms.fetch(a.teacher, row);
      terms.fetch_logits(x);
    } else {
      if (tok < 0) {
        write_padding<BT>(a, row);
        continue;
      }
      if (tok < a.V) token_logit = to_f32(x[tok]);
    }
    const float m = block_max<BT>(mp);
    const float d = sp == 0.f ? 0.f : (mp - m) * a.scale2;
    const float w = exp2_raw(d);
    const float s = block_sum<BT>(w * sp);
    float t = 0.f;
    if constexpr (ENT) t = block_sum<BT>(w * __builtin_fmaf(max_raw(d, -300.f), sp, tp));
    if constexpr (TOP) {
      auto emit = [&](int rank, uint64_t key) { emit_top(a, row, rank, key, m, s); };
      auto for_keys = [&](auto f) {
#pragma unroll
        for (int r = 0; r < R; ++r) f(keys[r]);
        for (int i = kCand + threadIdx.x; i < n; i += BT) f(key_at(i));
      };
      // at + 1 keys of a piece are at or above its at-th one: the `need` largest of those have k between them
      const int need = (a.top_k + at) / (at + 1), full = a.parts < 64 ? 1 : a.parts / 64;
      const uint64_t bound = block_bound(lds.top[0], lead, (need + full - 1) / full, full, 32);
      for_keys([&](uint64_t key) { push_key(lds.top[0], key, bound); });
      if (!emit_ranked(lds.top[0], a.top_k, emit)) {
        uint64_t last = ~0ull;
        for (int r = 0; r < a.top_k; ++r) {
          uint64_t best = 0;
          for_keys([&](uint64_t key) { best = key < last && key > best ? key : best; });
          last = block_max_key<BT>(best);
          if (threadIdx.x == 0) emit(r, last);
        }
      }
    }
    write_row<BT, ENT, DIST>(a, row, tok, token_logit, m, s, t, terms);
  }
}

static bool bad_shape(int64_t N, int64_t V, int64_t row_stride, int dtype) {
  return N < 0 || V < 1 || V > VAE_MAX_ROW || (N > 1 && row_stride < V) ||
         (dtype != VAE_F32 && dtype != VAE_BF16 && dtype != VAE_F16);
}
static int grid_for(int64_t items) { return (int)(items < kMaxGrid ? items : kMaxGrid); }

// Pieces of a row: with up to kFillRows rows a workgroup a row leaves compute units idle.  Four workgroups a compute unit
// are aimed at, of kPieceVecs vectors or more (1 x 131072 bf16: 5.2 us with 512 or 128, 6.1 with 2048).  The second launch
// has its price, about 3 us, 5 with alternatives, so short rows stay whole:
//   bf16, split against whole:  64 x 131072 7.9 / 14.9 us,  256 x 131072 15.8 / 19.6,  400 x 131072 24.1 / 21.5,
//     1 x 65536 5.4 / 6.0,  256 x 65536 10.8 / 10.8,  1 x 32768 5.3 / 4.3,  128 x 32768 7.5 / 6.3;
//   with 5 alternatives:  1 x 131072 10.0 / 13.6,  64 x 131072 13.9 / 19.3,  1 x 65536 10.2 / 8.9,  256 x 65536 16.5 / 14.4.
constexpr int64_t kFillRows = 256, kPieceVecs = 512, kSplitVecs = 8192, kSplitVecsTop = 16384;
struct Cut {
  int parts, part_vecs;
};
static Cut cut_rows(int64_t N, int64_t V, int64_t top_k, int dtype) {
  const int64_t vn = dtype == VAE_F32 ? 4 : 8;
  const int64_t nvec = (V + vn - 1) / vn;
  int64_t parts = 1;
  if (N <= kFillRows && V / vn >= (top_k ? kSplitVecsTop : kSplitVecs)) {
    parts = 4 * kFillRows / (N > 0 ? N : 1);
    const int64_t most = nvec / kPieceVecs;
    parts = parts < most ? parts : most;
    parts = parts < 1 ? 1 : (parts > kBlock ? kBlock : parts);
  }
  const int64_t per = (nvec + parts - 1) / parts;
  return {(int)((nvec + per - 1) / per), (int)per};
}

template <typename T, int BT, bool ENT, bool TOP, bool DIST>
static int fwd_launch(const FwdArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((token_fwd_kernel<T, BT, ENT, TOP, DIST>), dim3(grid_for(a.N * a.parts)), dim3(BT), 0, st, a);
  if (a.parts > 1)
    hipLaunchKernelGGL((token_join_kernel<T, kBlock, ENT, TOP, DIST>), dim3(grid_for(a.N)), dim3(kBlock), 0, st, a);
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
}
// A wave a row for rows of up to 512 vectors, and of up to 1024 where there are many: no barriers, and four or more rows a
// compute unit's worth of loads.  65536 x 4096 bf16: 82 us (6.5 TB/s) against 142 with a workgroup a row; 8192 x 8192:
// 24.4 against 25.2, but 512 x 8192: 5.9 against 4.7; 8192 x 16384: 48.7 against 45.2.  Beyond 48 alternatives the bound
// would take nearly every lane's maximum, the least of 64, and a quarter of the row with it (16384 x 2000 bf16, 64 of
// them: 320 us against 84 with a workgroup, which asks each wave for its 16 largest; 48 of them: 61 against 73).
template <typename T, bool DIST>
static int fwd_type(const FwdArgs& a, hipStream_t st) {
  const int64_t nvec = (a.V + VecOf<T>::n - 1) / VecOf<T>::n;
  const bool wave = a.parts == 1 && (nvec <= 512 || (nvec <= 1024 && a.N >= 2048)) && !(a.top_k > 48 && nvec >= 224);
#define VAE_FWD(E, K) (wave ? fwd_launch<T, 64, E, K, DIST>(a, st) : fwd_launch<T, kBlock, E, K, DIST>(a, st))
  if constexpr (DIST) return VAE_FWD(false, false);
  else {
    if (a.entropy) return a.top_k ? VAE_FWD(true, true) : VAE_FWD(true, false);
    return a.top_k ? VAE_FWD(false, true) : VAE_FWD(false, false);
  }
#undef VAE_FWD
}

// kl and stats; vae_distill_fwd (token_grad.hip) has checked the arguments
int distill_stats(const void* logits, int64_t row_stride, const Teacher& teacher, float temperature, float* kl,
                  float* stats, void* scratch, int64_t N, int64_t V, int dtype, hipStream_t stream) {
  const Cut cut = cut_rows(N, V, 0, dtype);
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
  const Cut c = cut_rows(N, V, top_k, dtype);
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
  const Cut cut = cut_rows(N, V, top_k, dtype);
  if (cut.parts > 1 && !scratch) return VAE_ERR_ARG;
  const FwdArgs a = {logits, row_stride, tokens, token_bytes, logp, entropy, stats, top_logp, top_ids, (int)top_k, N,
                     (int)V, cut.parts, cut.part_vecs, (char*)scratch, kLog2e, 1.0f, {}};
  VAE_BY_TYPE(dtype, return (fwd_type<T, false>(a, (hipStream_t)stream)));
  return VAE_ERR_ARG;
}

}  // extern "C"
