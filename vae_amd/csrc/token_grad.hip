// Gradients with respect to rows of logits [N, V]: of log probs, entropy and alternatives (token_logp_bwd), of the
// distillation KL (distill_bwd), and both losses together with their gradient in one pass (token_fused_kernel).  Formulas
// and the conventions for masks: token_row.hpp.
//
// Every one of them is   g_j = e_j (A + B d_j) + sum over a few entries (id, g) with id = j,   d = (x - m) c, e = 2^d:
//   tokens:   A = -(sum_i g_i + g_H (H - ln s)) / s,  B = -g_H ln2 / s,  entries: the token and the alternatives
//   teacher:  A = w / (tau s),  B = 0,  entries: (id_k, -w q_k / tau)
// The entries are owned by the thread whose vector holds them and added before the vector is stored: no atomics on the
// gradient, no second write, one rounding.
#include "token_row.hpp"

namespace vae {

// A piece's entries in LDS, each thread's own in a list.  No id comes twice, so the order of a list does not matter.
constexpr int kMaxEntries = VAE_MAX_TEACHER;
template <int BT>
struct Entries {
  int head[BT];
  int next[kMaxEntries], id[kMaxEntries];
  float g[kMaxEntries];

  // a barrier of the caller's stands between clear() and put(), and between put() and the lists' use
  __device__ __forceinline__ void clear(bool again) {
    if (again) lds_barrier();   // the row before this one has been read
    head[threadIdx.x] = -1;
  }
  template <typename T, int VN>
  __device__ __forceinline__ void put(int k, int id_k, float g_k, const RowCut<T, VN>& cut, int v0, int v1) {
    if (id_k < 0) return;
    const int off = id_k - cut.head;
    int owner = -1;
    if (off < 0) owner = id_k;                                      // RowCut::edge
    else if (off >= cut.nvec * VN) owner = 16 + off - cut.nvec * VN;
    else if (off / VN >= v0 && off / VN < v1) owner = (off / VN - v0) % BT;
    if (owner < 0) return;
    id[k] = id_k;
    g[k] = g_k;
    next[k] = atomicExch(&head[owner], k);
  }
};

// What a thread adds to its elements: one entry known to all, or (LIST) the workgroup's lists.
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
  Teacher teacher;
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
    for (int u = 0; u < U; ++u) p[u].load(in, byte + u * BT * P::kBytes);
  }
  __device__ __forceinline__ void mask() {       // what is not there counts as masked out
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((u + 1) * BT > nvec && (int)threadIdx.x + u * BT >= nvec) p[u].set_masked();
  }
  __device__ __forceinline__ void store(bool nts, int u, const float (&v)[VN]) const {
    int at = byte;
    asm volatile("" : "+v"(at));   // added up again: the loads' offsets are not kept in registers for it
    P::store(out, nts, at + u * BT * P::kBytes, v);
  }
  __device__ __forceinline__ void fill(bool nts, float value) const {
    float v[VN];
#pragma unroll
    for (int i = 0; i < VN; ++i) v[i] = value;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (any(u)) store(nts, u, v);
  }
};

// ---------------------------------------------------------------------------------------------------------------
// from given statistics: one read, one write, and bound by them.  A workgroup takes one piece of U vectors a thread, all
// loads in front of all stores: in a loop the loads of a turn wait for the stores of the turn before it.  4096 x 32768
// bf16: 87 us (6.1 TB/s read + written), with entropy too; 153 us with a loop over U = 4.  Distillation, 64 entries: 85.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int VN, int BT, int U, bool ENT, bool LIST, bool DIST>
__global__ __launch_bounds__(BT) void token_bwd_kernel(GradArgs a) {
  __shared__ struct {
    Entries<BT> entries[LIST ? 1 : 0];
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
    const bool bad = !DIST && tok >= a.V && (!a.glogp || a.g_scale != 0.f);   // the gradient of its NaN
    if (tok < 0 || s == 0.f || bad) {
      const float v = bad ? nan_f() : 0.f;
      piece.fill(a.nts, v);
      if (ei >= 0) gx[ei] = from_f32<T>(v);
      continue;
    }
    TeacherTerms<BT> terms;
    if constexpr (DIST) terms.fetch(a.teacher, row);
    piece.load();
    const float edge = ei >= 0 ? to_f32(x[ei]) : 0.f;
    Adds<T, VN, BT, LIST> adds;
    if constexpr (LIST) adds.lds = lds.entries;
    float A, B = 0.f;
    const float inv = 1.0f / s;
    if constexpr (DIST) {
      const float g0 = a.gmean ? a.gmean[0] * a.mean_scale : (a.gkl ? 0.f : a.mean_scale);
      const float w = ((a.gkl ? a.gkl[row] : 0.f) + g0) * a.inv_tau;
      A = w * inv;               // an id beyond the vocabulary: s is NaN
      lds.entries[0].clear(item != blockIdx.x);
      lds_barrier();
#pragma unroll
      for (int r = 0; r < TeacherTerms<BT>::R; ++r)
        lds.entries[0].put((int)threadIdx.x + r * BT, terms.id[r], -w * terms.q[r], cut, v0, v1);
      lds_barrier();
    } else {
      const float gt = a.tokens ? (a.glogp ? a.glogp[row / a.rows_per_g] * a.g_scale : a.g_scale) : 0.f;
      const bool inside = a.tokens && tok < a.V;
      float sum = gt;
      adds.one_id = inside ? (int)tok : -1;
      adds.one_g = gt;
      if constexpr (LIST) {
        for (int k = 0; k < a.top_k; ++k) sum += a.gtop[row * a.top_k + k];
        // the alternatives differ from each other; the token may be one of them
        lds.entries[0].clear(item != blockIdx.x);
        lds_barrier();
        bool other = true;
        for (int k = 0; k < a.top_k; ++k) other &= a.top_ids[row * a.top_k + k] != tok;
        for (int k = threadIdx.x; k <= a.top_k; k += BT) {
          const int id = k < a.top_k ? (int)a.top_ids[row * a.top_k + k] : (other ? adds.one_id : -1);
          const float g = k < a.top_k ? a.gtop[row * a.top_k + k] : 0.f;
          lds.entries[0].put(k, id, g + (id == adds.one_id ? gt : 0.f), cut, v0, v1);
        }
        lds_barrier();
      }
      if constexpr (ENT) {
        const float gh = a.gentropy[row];
        sum += gh * (a.entropy[row] - kLn2 * log2f(s));
        B = -gh * kLn2 * inv;
      }
      A = -sum * inv;
    }
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
// loss and gradient in one pass: a workgroup holds its row in registers, U vectors a thread, as every element's
// exponential against the thread's own maximum: one exponential an element (AGAIN: two), the gradient is a product.
// Bound by memory: 4096 x 131072 bf16 412 us (5.2 TB/s read + written), as a distillation too; 8144 x 65536 375 us (5.7);
// 16384 x 16384 181 us (5.9); two passes instead 525 (584 as a distillation), 553 and 268.  fp32: 4096 x
// 32768 192 us (5.6), 4096 x 65536 404 us (5.3), though 64 exponentials a thread beside the packets spill 60 bytes a lane (104
// with a teacher, 221 and 424 us; bf16 with a teacher 12 and 40).
// An exponential takes a register, 8 a 16-bit vector.  AGAIN: bf16 rows that do not fit so stay as their packets, 4
// registers a vector, and the gradient forms its exponentials again: 4096 x 131072 412 us, 401 with them kept in binary16,
// which lost bits of probabilities below 2^-29 of a thread's largest and left nothing of those below 2^-40.
// ---------------------------------------------------------------------------------------------------------------
template <typename T, int BT, int U, bool AGAIN, bool DIST>
__global__ __launch_bounds__(BT, 4) void token_fused_kernel(GradArgs a) {
  constexpr int VN = VecOf<T>::n;
  __shared__ struct {
    Entries<BT> entries[DIST ? 1 : 0];
  } lds;
  for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* x = (const T*)a.logits + row * a.row_stride;
    T* gx = (T*)a.glogits + row * (int64_t)a.V;
    const RowCut<T, VN> cut(x, a.V);
    const int ei = cut.edge(threadIdx.x);
    Piece<T, VN, BT, U> piece(x, gx, cut, 0, cut.nvec);
    int64_t tok = 0;
    int state = kRowFine;
    float token_logit = 0.f;
    if constexpr (DIST) {
      state = a.teacher.state[row];
    } else {
      tok = load_id(a.tokens, a.token_bytes, row);
      state = tok < 0 ? kRowEmpty : (tok >= a.V ? kRowBad : kRowFine);
      if (state == kRowFine) token_logit = to_f32(x[tok]);
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
    TeacherTerms<BT> terms;
    if constexpr (DIST) terms.fetch(a.teacher, row);
    piece.load();
    const float edge = ei >= 0 ? to_f32(x[ei]) : -INFINITY;
    if constexpr (DIST) {
      lds.entries[0].clear(row != blockIdx.x);
      terms.fetch_logits(x);
    }
    piece.mask();
    float mt = max_raw(edge, kLowest);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (piece.any(u)) {
        float v[VN];
        piece.p[u].get(v);
        mt = vec_max(v, mt);
      }
    float e[AGAIN ? 1 : U][VN];
    float s = exp2_raw((edge - mt) * a.scale2);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (piece.any(u)) {
        asm volatile("" : "+v"(piece.p[u].raw));   // unpack again: the packets, not their elements, stay in registers
        float v[VN];
        piece.p[u].get(v);
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          v[i] = exp2_raw((v[i] - mt) * a.scale2);
          s += v[i];
        }
        if constexpr (!AGAIN) {
#pragma unroll
          for (int i = 0; i < VN; ++i) e[u][i] = v[i];
        }
      }
    const float m = block_max<BT>(mt);
    float f = exp2_raw((mt - m) * a.scale2);       // from the thread's maximum to the row's
    // The entries between the two reductions, whose barriers they need: a wave's exponentials wait for its own packets
    // alone.
    Adds<T, VN, BT, DIST> adds;
    const float w = DIST ? a.mean_scale * a.inv_tau : a.g_scale;   // of p; the entries have the other sign
    if constexpr (DIST) {
      adds.lds = lds.entries;
      if constexpr (BT == 64) lds_barrier();       // block_max has none
#pragma unroll
      for (int r = 0; r < TeacherTerms<BT>::R; ++r)
        lds.entries[0].put((int)threadIdx.x + r * BT, terms.id[r], -w * terms.q[r], cut, 0, cut.nvec);
      if constexpr (BT == 64) lds_barrier();
    } else {
      adds.one_id = (int)tok;
      adds.one_g = -w;
    }
    s = block_sum<BT>(s * f);
    adds.prepare(cut, 0, cut.nvec);
    // in front of the gradient: behind it this would wait for the stores, loads and stores share a counter
    if constexpr (DIST) {
      const float kl = terms.kl(a.teacher.K, m, s, a.inv_tau);
      if (threadIdx.x == 0) a.out[row] = kl;
    } else if (threadIdx.x == 0) {
      a.out[row] = row_log_prob(token_logit, m, s, 1.0f);
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
        if constexpr (AGAIN) {
          asm volatile("" : "+v"(piece.p[u].raw));
          piece.p[u].get(v);
#pragma unroll
          for (int i = 0; i < VN; ++i) v[i] = A * exp2_raw((v[i] - m) * a.scale2);
        } else {
#pragma unroll
          for (int i = 0; i < VN; ++i) v[i] = f * e[u][i];
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
  // a wave a row where it fits (distillation of 65536 x 2048 bf16: 92 us, 146 with 256 threads; 1024: 58, 135)
  if (nvec <= 256) return bwd_launch<T, VN, 64, 4, ENT, LIST, DIST>(a, st);
  // U = 4 (65536 x 4096 bf16: 179 us; U = 8 192, U = 16 242).  Alternatives are looked through once a piece: twice as
  // long a piece for them (4096 x 32768, 8 of them: U = 4 114 us, U = 8 102; the teacher's come prepared: 87 and 91).
  return bwd_launch<T, VN, kBlock, LIST && !DIST ? 8 : 4, ENT, LIST, DIST>(a, st);
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

template <typename T, int BT, int U, bool AGAIN, bool DIST>
static int fused_launch(GradArgs a, hipStream_t st) {
  a.nts = (int64_t)sizeof(T) * a.N * a.V >= kNtStoreMinBytes;
  hipLaunchKernelGGL((token_fused_kernel<T, BT, U, AGAIN, DIST>), dim3(grid_for(a.N)), dim3(BT), 0, st, a);
  return launched();
}
// true when the one-pass kernel takes this call: the row fits a workgroup's registers, and there are rows enough.
// fp16 never: a stored gradient is of a mean, whose 1 / N is a subnormal of fp16.
template <typename T, bool DIST>
static bool fused_type(const GradArgs& a, hipStream_t st, int* rc) {
  if constexpr (DTypeCode<T>::value != VAE_F16) {
    constexpr int E = 64 / VecOf<T>::n, H = E / 2;   // vectors a thread: 64 or 32 elements
    const int64_t nvec = (int64_t)a.V / VecOf<T>::n;
    // AGAIN for bf16 only: an fp32 packet is as large as its exponentials
    constexpr int most = DTypeCode<T>::value == VAE_BF16 ? 16 : E;
    // AGAIN with few rows: two launches that cut the rows (64 x 131072 bf16: 19.1 us, 21.4 in one; 16 x 131072 17.9, 19.3;
    // but 100 x 131072: 25.4, 23.1; without AGAIN 16 x 65536 12.2, 10.7)
    if (!same_phase<T>(a) || nvec > 1024 * most || (a.N <= 64 && nvec > 1024 * E && most > E)) return false;
    // 32 elements a thread while 512 threads hold the row so: more waves in flight (32768 x 8192 bf16 179 us, 189 with
    // 64; 8192 x 16384 fp32 186, 213); 64 beyond, where 1024 threads of 32 wait for each other longer (8192 x 32768 bf16:
    // 193 us, 235 with 32)
    if (nvec <= 64 * H) *rc = fused_launch<T, 64, H, false, DIST>(a, st);
    else if (nvec <= 128 * H) *rc = fused_launch<T, 128, H, false, DIST>(a, st);
    else if (nvec <= 256 * H) *rc = fused_launch<T, 256, H, false, DIST>(a, st);
    else if (nvec <= 512 * H) *rc = fused_launch<T, 512, H, false, DIST>(a, st);
    else if (nvec <= 512 * E) *rc = fused_launch<T, 512, E, false, DIST>(a, st);
    else if (nvec <= 1024 * E) *rc = fused_launch<T, 1024, E, false, DIST>(a, st);
    else if constexpr (most > E) *rc = fused_launch<T, 1024, most, true, DIST>(a, st);
    return true;
  }
  return false;
}

static bool bad_teacher(int64_t K, float temperature) {
  // below 4.3e-39 its reciprocal leaves fp32's range
  return K < 1 || K > VAE_MAX_TEACHER || !(temperature > 4.3e-39f) || !(temperature < INFINITY);
}
static void set_temperature(GradArgs& a, float temperature) {
  a.scale2 = (float)(1.4426950408889634 / (double)temperature);
  a.inv_tau = (float)(1.0 / (double)temperature);
}

int token_nll_grad(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp, float* stats,
                   void* glogits, float grad_scale, void* scratch, int64_t N, int64_t V, int dtype,
                   hipStream_t stream) {
  int rc = VAE_ERR_ARG;
  ShortArgs sa = {logits, row_stride, tokens, token_bytes, N, (int)V, logp, nullptr, stats, nullptr, nullptr, 0,
                  glogits, nullptr, 1, -grad_scale, nullptr, nullptr, nullptr, 0};
  if (short_rows(sa, dtype, stream, &rc)) return rc;
  GradArgs a = {};
  a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
  a.scale2 = kLog2e; a.inv_tau = 1.0f;
  a.tokens = tokens; a.token_bytes = token_bytes; a.g_scale = grad_scale; a.out = logp; a.stats_out = stats;
  VAE_BY_TYPE(dtype, if (fused_type<T, false>(a, stream, &rc)) return rc);
  rc = vae_token_logp_fwd(logits, row_stride, tokens, token_bytes, logp, nullptr, stats, nullptr, nullptr, 0, scratch, N,
                          V, dtype, stream);
  if (rc != VAE_OK) return rc;
  return vae_token_logp_bwd(logits, row_stride, tokens, token_bytes, stats, nullptr, nullptr, 1, -grad_scale, nullptr,
                            nullptr, nullptr, 0, glogits, N, V, dtype, stream);
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

int vae_distill_bwd(const void* logits, int64_t row_stride, const float* teacher, int64_t K, float temperature,
                    const float* stats, const float* gkl, const float* gmean, float mean_scale, void* glogits,
                    int64_t N, int64_t V, int dtype, vae_stream_t stream) {
  if (bad_rows(N, V, row_stride, dtype) || bad_teacher(K, temperature)) return VAE_ERR_ARG;
  if (N == 0) return VAE_OK;
  if (!logits || !teacher || !stats || !glogits) return VAE_ERR_ARG;
  GradArgs a = {};
  a.teacher = teacher_of(teacher, N, K);
  a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
  a.stats_in = stats; a.gkl = gkl; a.gmean = gmean; a.mean_scale = mean_scale;
  set_temperature(a, temperature);
  VAE_BY_TYPE(dtype, return (bwd_type<T, true>(a, (hipStream_t)stream)));
  return VAE_ERR_ARG;
}

int vae_distill_fwd(const void* logits, int64_t row_stride, const void* t_logits, int64_t t_stride, int t_dtype,
                    const void* t_ids, int64_t id_stride, int id_bytes, int64_t K, float temperature, float* teacher,
                    float* kl, float* mean, float mean_scale, float* stats, void* glogits, void* scratch, int64_t N,
                    int64_t V, int dtype, vae_stream_t stream) {
  if (bad_rows(N, V, row_stride, dtype) || bad_teacher(K, temperature) || !type_ok(t_dtype) ||
      (id_bytes != 4 && id_bytes != 8) || (N > 1 && (t_stride < K || id_stride < K)))
    return VAE_ERR_ARG;
  if (N == 0) return mean ? vae_row_sums(nullptr, mean_scale, mean, 1, 0, VAE_F32, stream) : VAE_OK;
  if (!logits || !t_logits || !t_ids || !teacher || !kl || (glogits && !stats)) return VAE_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (vae_token_scratch_bytes(N, V, 0, dtype) && !scratch) return VAE_ERR_ARG;
  int rc = prepare_teacher(t_logits, t_stride, t_dtype, t_ids, id_stride, id_bytes, K, temperature, teacher, N, V, st);
  if (rc != VAE_OK) return rc;
  GradArgs a = {};
  a.teacher = teacher_of(teacher, N, K);
  bool done = false;
  if (glogits) {
    a.logits = logits; a.row_stride = row_stride; a.glogits = glogits; a.N = N; a.V = (int)V;
    a.mean_scale = mean_scale; a.out = kl; a.stats_out = stats;
    set_temperature(a, temperature);
    VAE_BY_TYPE(dtype, done = fused_type<T, true>(a, st, &rc));
  }
  if (!done) {
    rc = distill_stats(logits, row_stride, a.teacher, temperature, kl, stats, scratch, N, V, dtype, st);
    if (rc == VAE_OK && glogits)
      rc = vae_distill_bwd(logits, row_stride, teacher, K, temperature, stats, nullptr, nullptr, mean_scale, glogits, N,
                           V, dtype, stream);
  }
  if (rc != VAE_OK || !mean) return rc;
  return vae_row_sums(kl, mean_scale, mean, 1, N, VAE_F32, stream);
}

}  // extern "C"
