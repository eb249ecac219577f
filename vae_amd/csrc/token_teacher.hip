// The teacher's side of a distillation, once per call: q = softmax(y / tau) over the entries that are there (id >= 0,
// logit > -inf), ln q, and what comes twice merged, so that the kernels over the vocabulary find each id once.  A wave a
// row, no barrier: K entries are 2 KB at most.  Prepared here and not in those kernels: there the chain of loads and
// reductions stood in front of every row (4096 x 131072 bf16 with K = 64: 531 us against 423 us of the loss that has no
// teacher; 8192 x 32768: 435 against 182).  65536 rows of 64 entries: 27 us.  1, 2 or 4 entries a lane as
// K asks (the whole call for 65536 x 1024 with 64 entries: 117 us, 131 with 4 for all).
#include "token_row.hpp"

namespace vae {

constexpr int kSlots = 1024;   // 64 ids leave about 2 pairs in one slot, 256 about 32
static_assert(VAE_MAX_ROW <= 1 << 24 && VAE_MAX_TEACHER <= 256, "an id and its place share 32 bits");
__device__ __forceinline__ uint32_t slot_of(int id) { return (uint32_t)id * 2654435761u >> 22; }

// LDS that only one wave uses: its lanes' writes in front of its lanes' reads, without a barrier of the workgroup (the
// waves of one take different numbers of rounds)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int R>   // entries a lane
__global__ __launch_bounds__(kBlock) void distill_teacher_kernel(const void* __restrict__ logits, int64_t stride, int dtype,
                                                                 const void* __restrict__ ids, int64_t id_stride,
                                                                 int id_bytes, int K, float inv_tau, float scale2,
                                                                 int* __restrict__ state, int* __restrict__ id_out,
                                                                 float* __restrict__ q_out, float* __restrict__ logq_out,
                                                                 int64_t N, int V) {
  __shared__ uint32_t slots[kBlock / 64][kSlots];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t row = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6); row < N;
       row += (int64_t)gridDim.x * (kBlock / 64)) {
    float y[R], q[R], logq[R], m = kLowest;
    int id[R];
    bool bad = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = lane + 64 * r;
      y[r] = -INFINITY;
      id[r] = -1;
      if (k < K) {
        const int64_t i = load_id(ids, id_bytes, row * id_stride + k);
        bad |= i >= V;
        if (i >= 0 && i < V) {
          id[r] = (int)i;
          y[r] = load_any(logits, dtype, row * stride + k);
        }
      }
      m = max_raw(m, y[r]);
    }
    m = group_max(m, 64);
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      q[r] = id[r] >= 0 ? exp2_raw((y[r] - m) * scale2) : 0.f;
      if (q[r] == 0.f) id[r] = -1;
      s += q[r];
    }
    s = group_sum(s, 64);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      q[r] /= s;
      logq[r] = row_log_prob(y[r], m, s, inv_tau);
    }
    // Which ids come twice: every entry writes (id, its place) into the slot of its id's hash and reads the slot back.  Its
    // own: it is the first to stand for its id.  The same id at another place: it is a second one.  Another id: once more,
    // without those that are settled.  Every round settles each slot's writer, so it ends.  (An entry compared with every
    // other one: 194 us for 65536 rows of 64 entries.)
    bool todo[R], again[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      todo[r] = id[r] >= 0;
      again[r] = false;
    }
    for (;;) {
      bool any = false;
#pragma unroll
      for (int r = 0; r < R; ++r) any |= todo[r];
      if (__ballot(any) == 0) break;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (todo[r])
          __hip_atomic_store(&slots[wave][slot_of(id[r])], (uint32_t)id[r] | (uint32_t)(lane + 64 * r) << 24,
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
      wave_fence();
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (todo[r]) {
          const uint32_t w = __hip_atomic_load(&slots[wave][slot_of(id[r])], __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_WAVEFRONT);
          todo[r] = (w & 0xffffffu) != (uint32_t)id[r];
          again[r] = !todo[r] && (int)(w >> 24) != lane + 64 * r;
        }
      wave_fence();
    }
    // one id's entries into the first of them: the sum of q, and of q ln q, in the entries' order
#pragma unroll
    for (int r0 = 0; r0 < R; ++r0)
      for (uint64_t left = __ballot(again[r0]); left != 0; left = __ballot(again[r0])) {
        const int common = __builtin_amdgcn_readlane(id[r0], __ffsll((unsigned long long)left) - 1);
        float qs = 0.f, ql = 0.f;
        int first = -1;
#pragma unroll
        for (int r = 0; r < R; ++r)
          for (uint64_t all = __ballot(id[r] == common); all != 0; all &= all - 1) {
            const int l = __ffsll((unsigned long long)all) - 1;
            const float oq = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, q[r]), l));
            const float ol = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, logq[r]), l));
            qs += oq;
            ql = __builtin_fmaf(oq, ol, ql);
            first = first < 0 ? l + 64 * r : first;
          }
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (id[r] == common) {
            again[r] = false;
            if (lane + 64 * r == first) {
              q[r] = qs;
              logq[r] = ql / qs;   // weighted: q (ln q - ln p) of the merged entry is their sum
            } else {
              id[r] = -1;
            }
          }
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = lane + 64 * r;
      if (k >= K) continue;
      id_out[row * K + k] = id[r];
      q_out[row * K + k] = q[r];
      logq_out[row * K + k] = logq[r];
    }
    const bool any_bad = __ballot(bad) != 0 || s != s;   // NaN or +inf among the teacher's: no distribution either
    if (lane == 0) state[row] = any_bad ? kRowBad : (s == 0.f ? kRowEmpty : kRowFine);
  }
}

int prepare_teacher(const void* t_logits, int64_t t_stride, int t_dtype, const void* t_ids, int64_t id_stride,
                    int id_bytes, int64_t K, float temperature, float* teacher, int64_t N, int64_t V,
                    hipStream_t stream) {
  const Teacher t = teacher_of(teacher, N, K);
  const int64_t blocks = (N + kBlock / 64 - 1) / (kBlock / 64);
  const int grid = (int)(blocks < kMaxGrid ? blocks : kMaxGrid);
  const float inv_tau = (float)(1.0 / (double)temperature);
  const float scale2 = (float)(1.4426950408889634 / (double)temperature);
  const auto kernel = K <= 64    ? distill_teacher_kernel<1>
                      : K <= 128 ? distill_teacher_kernel<2>
                                 : distill_teacher_kernel<4>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kBlock), 0, stream, t_logits, t_stride, t_dtype, t_ids, id_stride,
                     id_bytes, (int)K, inv_tau, scale2, const_cast<int*>(t.state), const_cast<int*>(t.id),
                     const_cast<float*>(t.q), const_cast<float*>(t.logq), N, (int)V);
  return hipGetLastError() == hipSuccess ? VAE_OK : VAE_ERR_LAUNCH;
}

}  // namespace vae

extern "C" {

size_t vae_distill_teacher_floats(int64_t N, int64_t K) {
  return N < 0 || K < 1 || K > VAE_MAX_TEACHER ? 0 : (size_t)N * (1 + 3 * (size_t)K);
}

}  // extern "C"
