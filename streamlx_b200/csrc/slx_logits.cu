// Logit processing of a batch (sm_100a): penalties for repeated tokens,
// biases, grammar mask and the greedy pick in one launch.
#include <cooperative_groups.h>

#include "slx_kernels.cuh"

namespace slx {

namespace cg = cooperative_groups;

// What the rules say about one id, in one shared-memory word:
//   bit 31       the id stands in the row's history
//   bits 18..30  1 + the last bias entry of the row that names it (0: none)
//   bits 0..17   its occurrences in the row's output
constexpr uint32_t kSeen = 0x80000000u;
constexpr int kBiasShift = 18;
constexpr int kMaxBias = 8191;
constexpr uint32_t kCountMask = (1u << kBiasShift) - 1;

constexpr int kLogitCluster = 8;
constexpr int kLogitThreads = 512;
constexpr int kLogitSpan = 24576;  // ids per CTA and pass: 96 KB of words

struct Pick {  // best value so far and its id
  double v;
  int i;
  SLX_DEV void take(double x, int id) {
    if (x != x) x = -INFINITY;  // a NaN counts as -inf
    if (x > v || (x == v && id < i)) {
      v = x;
      i = id;
    }
  }
};

// A cluster of 8 CTAs per row, each with a slice of the vocabulary: zero a
// word per id, note the biases and the history in it, then one pass over the
// logits.  Ids without a word (nearly all) are copied; the others are
// computed in fp64, so picks between neighbouring values do not depend on
// the rounding of an intermediate.
template <typename T>
__global__ void __cluster_dims__(kLogitCluster, 1, 1)
    __launch_bounds__(kLogitThreads) k_logits(const LogitArgs a) {
  extern __shared__ uint32_t s_word[];
  __shared__ double s_v[kLogitThreads / 32];
  __shared__ int s_i[kLogitThreads / 32];
  __shared__ double c_v[kLogitCluster];
  __shared__ int c_i[kLogitCluster];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int b = blockIdx.x / kLogitCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  // CTA 0's shared memory is written by the others at the end: a CTA that
  // has passed the matching wait knows that CTA 0 runs
  cluster.barrier_arrive();
  pdl_wait_primary();
  const slx_logit_rules& R = a.r;
  int n_hist = 0, n_prompt = 0, bias0 = 0, bias1 = 0;
  bool bad = false;
  if (R.history) {
    n_hist = R.n_history[b];
    n_prompt = R.n_prompt ? R.n_prompt[b] : 0;
    bad = n_hist < 0 || n_hist > R.history_stride || n_prompt < 0 || n_prompt > n_hist;
    n_hist = min(max(n_hist, 0), R.history_stride);
    n_prompt = min(max(n_prompt, 0), n_hist);
  }
  if (R.bias_ids) {
    bias0 = R.bias_start[b];
    bias1 = R.bias_start[b + 1];
    bad |= bias0 < 0 || bias1 < bias0 || bias1 > R.n_bias || bias1 - bias0 > kMaxBias;
    bias0 = min(max(bias0, 0), R.n_bias);
    bias1 = min(max(bias1, bias0), R.n_bias);
    bias1 = min(bias1, bias0 + kMaxBias);
  }
  if (bad && rank == 0 && tid == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
  const bool words = n_hist > 0 || bias1 > bias0;
  const double rep = R.repetition ? (double)R.repetition[b] : 1.0;
  const double freq = R.frequency ? (double)R.frequency[b] : 0.0;
  const double pres = R.presence ? (double)R.presence[b] : 0.0;
  const T* x_row = reinterpret_cast<const T*>(a.logits) + (size_t)b * a.V;
  T* o_row = a.out ? reinterpret_cast<T*>(a.out) + (size_t)b * a.V : nullptr;
  const int32_t* hist = R.history ? R.history + (size_t)b * R.history_stride : nullptr;
  const uint32_t* mask = R.mask ? R.mask + (size_t)b * R.mask_stride : nullptr;
  Pick best = {-INFINITY, 0x7fffffff};
  const long long slice = ((a.V + kLogitCluster - 1LL) / kLogitCluster + 31) / 32 * 32;
  const long long end = min((long long)a.V, (rank + 1) * slice);
  for (long long lo = rank * slice; lo < end; lo += kLogitSpan) {
    const int v0 = (int)lo, n = (int)min((long long)kLogitSpan, end - lo);
    if (words) {
      __syncthreads();
      for (int i = tid; i < n; i += kLogitThreads) s_word[i] = 0;
      __syncthreads();
      for (int e = bias0 + tid; e < bias1; e += kLogitThreads) {
        const long long at = (long long)R.bias_ids[e] - v0;
        if (at >= 0 && at < n)
          atomicMax(&s_word[at], (uint32_t)(e - bias0 + 1) << kBiasShift);
      }
      __syncthreads();
      for (int e = tid; e < n_hist; e += kLogitThreads) {
        const long long at = (long long)hist[e] - v0;
        if (at >= 0 && at < n) {
          atomicOr(&s_word[at], kSeen);
          if (e >= n_prompt) atomicAdd(&s_word[at], 1u);
        }
      }
      __syncthreads();
    }
    for (int i = tid; i < n; i += kLogitThreads) {
      const int id = v0 + i;
      const bool ok = !mask || (mask[id >> 5] >> (id & 31) & 1u);
      T raw = x_row[id];
      float xf;
      if constexpr (sizeof(T) == 2) xf = bf16_to_f32(raw); else xf = raw;
      const uint32_t w = words ? s_word[i] : 0u;
      double x = xf;
      if (w) {
        if (w & kSeen) x = x > 0.0 ? x / rep : x * rep;
        const uint32_t c = w & kCountMask;
        if (c) x = __dsub_rn(__dsub_rn(x, __dmul_rn(freq, (double)c)), pres);
        const int e = (int)((w & ~kSeen) >> kBiasShift);
        if (e) x = __dadd_rn(x, (double)R.bias_values[bias0 + e - 1]);
        if constexpr (sizeof(T) == 2) raw = f32_to_bf16((float)x); else raw = (float)x;
      }
      if (!ok) {
        if constexpr (sizeof(T) == 2) raw = 0xff80u; else raw = -INFINITY;
      } else {
        best.take(x, id);
      }
      if (o_row) o_row[id] = raw;
    }
  }
  cluster.barrier_wait();
  if (!a.pick) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double v = __shfl_xor_sync(0xffffffffu, best.v, o);
    const int i = __shfl_xor_sync(0xffffffffu, best.i, o);
    best.take(v, i);
  }
  if (lane == 0) {
    s_v[warp] = best.v;
    s_i[warp] = best.i;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLogitThreads / 32; ++w) best.take(s_v[w], s_i[w]);
    *cluster.map_shared_rank(&c_v[rank], 0) = best.v;
    *cluster.map_shared_rank(&c_i[rank], 0) = best.i;
  }
  cluster.sync();
  if (rank == 0 && tid == 0) {
    best = {c_v[0], c_i[0]};
    for (int r = 1; r < kLogitCluster; ++r) best.take(c_v[r], c_i[r]);
    a.pick[b] = best.i < a.V ? best.i : -1;
  }
}

int launch_logits(const LogitArgs& a, bool f32, cudaStream_t s) {
  static PerDevice configured;
  std::atomic<int>& slot = configured.here();
  if (!slot.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(k_logits<uint16_t>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kLogitSpan * 4) != cudaSuccess ||
        cudaFuncSetAttribute(k_logits<float>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kLogitSpan * 4) != cudaSuccess)
      return SLX_ERR_CUDA;
    slot.store(1, std::memory_order_relaxed);
  }
  if (a.T > 0x7fffffff / kLogitCluster) return SLX_ERR_UNSUPPORTED;
  const long long slice = ((a.V + kLogitCluster - 1LL) / kLogitCluster + 31) / 32 * 32;
  const bool words = a.r.history || a.r.bias_ids;
  const size_t smem = words ? (size_t)(slice < kLogitSpan ? slice : kLogitSpan) * 4 : 0;
  const dim3 grid((unsigned)a.T * kLogitCluster);
  const cudaError_t e =
      f32 ? launch_k(k_logits<float>, grid, dim3(kLogitThreads), smem, s, a)
          : launch_k(k_logits<uint16_t>, grid, dim3(kLogitThreads), smem, s, a);
  return e == cudaSuccess ? SLX_OK : SLX_ERR_CUDA;
}

}  // namespace slx
