// What the token kernels (token.hip, token_grad.hip) share: a row of logits over a vocabulary, its softmax statistics,
// the ids that index it and the teacher's entries.  No reference counterpart: the reference's likelihoods are Bernoulli,
// Gaussian and the discretized logistic (abstract_vae.py:461-471); this is the categorical one.
//
// Statistics of a row x[V] at scale c = log2(e) / temperature:  m = max x,  s = sum 2^((x - m) c).
//   p_j = 2^((x_j - m) c) / s,   ln p_j = ln2 ((x_j - m) c - log2 s).
// The difference is formed before it is scaled: x = m gives exactly 1, and a row whose maximum is the type's lowest
// value (a mask written with it) does not overflow.  An all -inf row has s = 0 and no distribution: log p = -inf,
// entropy 0, gradient 0.  A NaN or +inf logit makes s NaN and with it everything the row returns.
#pragma once
#include "common.hpp"
#include "../../include/vae_amd.h"

namespace vae {

constexpr int kMaxGrid = 1 << 20;  // blocks of a launch; items beyond are grid-strided

// ids come as int32 or int64
__device__ __forceinline__ int64_t load_id(const void* __restrict__ ids, int id_bytes, int64_t i) {
  return id_bytes == 4 ? (int64_t) reinterpret_cast<const int32_t*>(ids)[i] : reinterpret_cast<const int64_t*>(ids)[i];
}
__device__ __forceinline__ float load_any(const void* __restrict__ p, int dtype, int64_t i) {
  if (dtype == VAE_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == VAE_BF16) return to_f32(reinterpret_cast<const bf16_t*>(p)[i]);
  return to_f32(reinterpret_cast<const f16_t*>(p)[i]);
}

// the least value a statistic is taken against: -inf would make x - m NaN
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float nan_f() { return __builtin_nanf(""); }
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// ln p of a value with statistics (m, s); s == 0: an empty row.  In natural units: x - m of the type's range does not
// overflow here, times log2(e) it could.
__device__ __forceinline__ float row_log_prob(float x, float m, float s, float inv_tau) {
  return s == 0.f ? -INFINITY : (x - m) * inv_tau - kLn2 * log2f(s);
}

// (value, index) as one sortable integer: larger value first, then the lower index; a NaN is below everything
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 and +0 are one value
  return x != x ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  const uint32_t o = order_bits(x);
  return o ? ((uint64_t)o << 32) | (uint32_t)(~index) : 0;  // 0: no entry
}
__device__ __forceinline__ float key_value(uint64_t key) { return order_value((uint32_t)(key >> 32)); }
__device__ __forceinline__ int64_t key_index(uint64_t key) { return (int64_t)(uint32_t)~(uint32_t)key; }

// Sum / max over a workgroup of BT threads, in a fixed order; every thread gets the result.  Uniform control flow.
template <int BT>
__device__ __forceinline__ float block_sum(float v) {
  v = group_sum(v, 64);
  if constexpr (BT > 64) {
    __shared__ float lds[BT / 64];
    lds_barrier();  // the readers of the last one are done
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    lds_barrier();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < BT / 64; ++w) v += lds[w];
  }
  return v;
}
template <int BT>
__device__ __forceinline__ float block_max(float v) {
  v = group_max(v, 64);
  if constexpr (BT > 64) {
    __shared__ float lds[BT / 64];
    lds_barrier();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    lds_barrier();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < BT / 64; ++w) v = max_raw(v, lds[w]);
  }
  return v;
}
template <int BT>
__device__ __forceinline__ uint64_t block_max_key(uint64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  if constexpr (BT > 64) {
    __shared__ uint64_t lds[BT / 64];
    lds_barrier();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    lds_barrier();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < BT / 64; ++w) v = lds[w] > v ? lds[w] : v;
  }
  return v;
}

// A row as a workgroup reads it: up to VN - 1 scalars in front of the first 16-byte boundary (threads 0..7 hold one
// each), `nvec` whole vectors, up to VN - 1 scalars behind them (threads 16..23).  Nothing outside the row is touched,
// whatever its alignment.  VN == 1: every element is a "vector" of its own.
template <typename T, int VN>
struct RowCut {
  int head, nvec, tail;
  __device__ __forceinline__ RowCut(const T* row, int V) {
    if constexpr (VN == 1) {
      head = tail = 0;
      nvec = V;
    } else {
      const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
      head = off ? VN - off : 0;
      head = head < V ? head : V;
      nvec = (V - head) / VN;
      tail = V - head - nvec * VN;
    }
  }
  // the scalar that thread `tid` holds, or -1
  __device__ __forceinline__ int edge(int tid) const {
    if (tid < head) return tid;
    if (tid >= 16 && tid < 16 + tail) return head + nvec * VN + (tid - 16);
    return -1;
  }
  __device__ __forceinline__ int index(int vec) const { return head + vec * VN; }
};

// A run of memory behind a buffer descriptor: the base and the length sit in scalar registers, a lane brings a 32-bit byte
// offset, and the hardware checks that offset against the length: a load beyond it returns zeros and a store beyond it is
// dropped, without a branch or a predicate.  The check covers the LANE's offset alone, not the instruction's scalar one, so
// whatever may lie beyond the run is addressed by the lane's offset.
struct Buffer {
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ Buffer(const void* base, int bytes)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000)) {}
};
constexpr int kNonTemporal = 2;   // cache policy operand of the buffer instructions

// Raw 16-byte packet of a row and its elements as floats.
template <typename T, int VN>
struct Packet {
  typedef uint32_t Raw __attribute__((ext_vector_type(4)));
  static constexpr int kBytes = 16;
  Raw raw;
  // `inside` is a scalar offset: lane_byte + inside is known to be within the run.  NT: not read again
  template <bool NT = true>
  __device__ __forceinline__ void load(const Buffer& b, int lane_byte, int inside = 0) {
    raw = __builtin_amdgcn_raw_buffer_load_b128(b.rsrc, lane_byte, inside, NT ? kNonTemporal : 0);
  }
  __device__ __forceinline__ void set_masked() {   // every element -inf
    const uint32_t inf = sizeof(T) == 4 ? 0xff800000u : (DTypeCode<T>::value == 2 ? 0xfc00fc00u : 0xff80ff80u);
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = inf;
  }
  __device__ __forceinline__ void get(float (&v)[VN]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(raw[i]);
      } else if constexpr (DTypeCode<T>::value == 2) {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(raw[i] & 0xffffu));
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(raw[i] >> 16));
      } else {
        v[2 * i] = __uint_as_float(raw[i] << 16);
        v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ static void store(const Buffer& b, bool nts, int lane_byte, const float (&v)[VN]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) r[i] = __float_as_uint(v[i]);
      else r[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    if (nts) __builtin_amdgcn_raw_buffer_store_b128(r, b.rsrc, lane_byte, 0, kNonTemporal);
    else __builtin_amdgcn_raw_buffer_store_b128(r, b.rsrc, lane_byte, 0, 0);
  }
};
// rows whose gradient is not aligned as they are: element by element
template <typename T>
struct Packet<T, 1> {
  static constexpr int kBytes = sizeof(T);
  T raw;
  template <bool NT = true>
  __device__ __forceinline__ void load(const Buffer& b, int lane_byte) {
    if constexpr (sizeof(T) == 4) raw = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b.rsrc, lane_byte, 0, 0));
    else raw.bits = __builtin_amdgcn_raw_buffer_load_b16(b.rsrc, lane_byte, 0, 0);
  }
  __device__ __forceinline__ void set_masked() { raw = from_f32<T>(-INFINITY); }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_f32(raw); }
  __device__ __forceinline__ static void store(const Buffer& b, bool, int lane_byte, const float (&v)[1]) {
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[0]), b.rsrc, lane_byte, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(from_f32<T>(v[0]).bits, b.rsrc, lane_byte, 0, 0);
  }
};
template <int VN>
__device__ __forceinline__ float vec_max(const float (&v)[VN], float m) {
  if constexpr (VN == 1) return max_raw(v[0], m);
#pragma unroll
  for (int i = 0; i + 1 < VN; i += 2) m = max3_raw(v[i], v[i + 1], m);
  return m;
}

// The teacher's entries as prepare_teacher (token_teacher.hip) leaves them: per row a state, and K entries of
// id (-1: none), q and ln q; entries of one id are merged into the first of them.
enum { kRowFine = 0, kRowEmpty = 1, kRowBad = 2 };  // nothing there | an id beyond the vocabulary, a NaN or +inf logit
struct Teacher {
  const int* state;       // [N]
  const int* id;          // [N, K]
  const float *q, *logq;  // [N, K]
  int K;
};
inline Teacher teacher_of(const float* buf, int64_t N, int64_t K) {
  Teacher t;
  t.state = reinterpret_cast<const int*>(buf);
  t.id = t.state + N;
  t.q = buf + N + N * K;
  t.logq = t.q + N * K;
  t.K = (int)K;
  return t;
}
int prepare_teacher(const void* t_logits, int64_t t_stride, int t_dtype, const void* t_ids, int64_t id_stride,
                    int id_bytes, int64_t K, float temperature, float* teacher, int64_t N, int64_t V, hipStream_t stream);
// kl [N] and stats [N, 2] of a distillation (token.hip); the arguments have been checked
int distill_stats(const void* logits, int64_t row_stride, const Teacher& teacher, float temperature, float* kl,
                  float* stats, void* scratch, int64_t N, int64_t V, int dtype, hipStream_t stream);
// logp and stats together with glogits = grad_scale * d(-logp) / d logits (token_grad.hip); checked
int token_nll_grad(const void* logits, int64_t row_stride, const void* tokens, int token_bytes, float* logp, float* stats,
                   void* glogits, float grad_scale, void* scratch, int64_t N, int64_t V, int dtype, hipStream_t stream);
// Each thread's entries of a row, asked for in three steps so that nobody waits: the entries in front of the row's
// packets, the student's logits there when the ids have come, the KL when the row's statistics are known.
template <int BT>
struct TeacherTerms {
  static constexpr int R = (VAE_MAX_TEACHER + BT - 1) / BT;
  int id[R];
  float q[R], logq[R], x[R];
  __device__ __forceinline__ void fetch(const Teacher& t, int64_t row) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = threadIdx.x + r * BT;
      const bool has = k < t.K;
      id[r] = has ? t.id[row * t.K + k] : -1;
      q[r] = has ? t.q[row * t.K + k] : 0.f;
      logq[r] = has ? t.logq[row * t.K + k] : 0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void fetch_logits(const T* __restrict__ logits) {
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = id[r] >= 0 ? to_f32(logits[id[r]]) : 0.f;
  }
  // the row's KL, in thread 0
  __device__ __forceinline__ float kl(int K, float m, float s, float inv_tau) const {
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (id[r] >= 0) v += q[r] * (logq[r] - row_log_prob(x[r], m, s, inv_tau));
    return K <= 64 ? group_sum(v, 64) : block_sum<BT>(v);   // up to 64 entries are the first wave's: no barrier
  }
};

// Short rows (token_short.hip): everything that is asked of a row from one reading of it.  False: the rows are too long
// for it, nothing was launched.
struct ShortArgs {
  const void* logits;
  int64_t row_stride;
  const void* tokens;
  int token_bytes;
  int64_t N;
  int V;
  float *logp, *entropy, *stats, *top_logp;        // each may be NULL
  int64_t* top_ids;
  int top_k;
  void* glogits;                                   // NULL: no gradient
  const float* glogp;
  int64_t rows_per_g;
  float g_scale;
  const float *gentropy, *gtop;
  const int64_t* gtop_ids;
  int gtop_k;
};
bool short_rows(const ShortArgs& a, int dtype, hipStream_t st, int* rc);

#define VAE_BY_TYPE(dtype_, ...)                                        \
  switch (dtype_) {                                                     \
    case VAE_F32: { using T = float; __VA_ARGS__; } break;              \
    case VAE_BF16: { using T = bf16_t; __VA_ARGS__; } break;            \
    case VAE_F16: { using T = f16_t; __VA_ARGS__; } break;              \
  }

}  // namespace vae
