// Logit processing of a batch (sm_100a): penalties for repeated tokens,
// biases, grammar mask and the greedy pick in one launch.
#include <cooperative_groups.h>

#include "slx_kernels.cuh"

namespace slx {

namespace cg = cooperative_groups;

// What the rules say about one id, in one shared-memory word:
//   bit 31       the id stands in the row's prompt
//   bits 18..30  1 + the last bias entry of the row that names it (0: none)
//   bits 0..17   its occurrences in the row's output
constexpr uint32_t kPrompt = 0x80000000u;
constexpr int kBiasShift = 18;
constexpr int kMaxBias = 8191;
constexpr uint32_t kCountMask = (1u << kBiasShift) - 1;

constexpr int kLogitCluster = 8;
constexpr int kLogitThreads = 512;
// 8-id vectors per thread and pass (registers: 20 and 24 for the logits)
template <typename T>
constexpr int kLogitVecs = sizeof(T) == 2 ? 5 : 3;
template <typename T>
constexpr int kLogitSpan = kLogitVecs<T> * kLogitThreads * 8;  // ids per CTA and pass

// Touched ids a pass lists; where there are more, the words are searched.
constexpr int kLogitList = 4096;

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

SLX_DEV float to_f32(uint16_t v) { return bf16_to_f32(v); }
SLX_DEV float to_f32(float v) { return v; }
SLX_DEV void from_f32(uint16_t* p, float x) { *p = f32_to_bf16(x); }
SLX_DEV void from_f32(float* p, float x) { *p = x; }

template <typename T>
struct Raw8;  // eight logits as loaded
template <>
struct Raw8<uint16_t> {
  uint32_t w[4];
  SLX_DEV float get(int j) const { return j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]); }
  SLX_DEV uint16_t bits(int j) const {
    const uint32_t lo = j & 2 ? w[1] : w[0], hi = j & 2 ? w[3] : w[2], x = j & 4 ? hi : lo;
    return (uint16_t)(j & 1 ? x >> 16 : x);
  }
  SLX_DEV void put(int j, uint16_t b) {
    w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | ((uint32_t)b << 16) : (w[j / 2] & 0xffff0000u) | b;
  }
  // -inf wherever the bit of `keep` is clear
  SLX_DEV void mask(uint32_t keep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = keep >> 2 * i;
      const uint32_t m = ((b & 1u) | (b & 2u) << 15) * 0xffffu;
      w[i] = (w[i] & m) | (0xff80ff80u & ~m);
    }
  }
  SLX_DEV float top() const {  // the greatest, NaN below everything
    auto max2 = [](uint32_t a, uint32_t b) {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                       *reinterpret_cast<const __nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    };
    const uint32_t m = max2(max2(w[0], w[1]), max2(w[2], w[3]));
    return fmaxf(fmaxf(bf16_lo(m), bf16_hi(m)), -INFINITY);
  }
  SLX_DEV void load(const uint16_t* p) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
  SLX_DEV void store(uint16_t* p) const {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
  SLX_DEV void load1(int j, const uint16_t* p) { put(j, *p); }
  SLX_DEV void store1(int j, uint16_t* p) const {
    *p = bits(j);
  }
};
template <>
struct Raw8<float> {
  float f[8];
  SLX_DEV float get(int j) const { return f[j]; }
  SLX_DEV float bits(int j) const {
    float x = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) x = i == j ? f[i] : x;
    return x;
  }
  SLX_DEV void mask(uint32_t keep) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!(keep >> j & 1)) f[j] = -INFINITY;
  }
  SLX_DEV float top() const {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, f[j]);
    return m;
  }
  SLX_DEV void load(const float* p) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
    const float4 b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  SLX_DEV void store(float* p) const {
    __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(f[4], f[5], f[6], f[7]));
  }
  SLX_DEV void load1(int j, const float* p) { f[j] = *p; }
  SLX_DEV void store1(int j, float* p) const { *p = f[j]; }
};

// Order of the picks as integers: greater values have greater keys.
SLX_DEV uint64_t pick_key(double v) {
  const long long b = __double_as_longlong(v + 0.0);  // -0 is 0
  return (uint64_t)(b < 0 ? ~b : b ^ (long long)0x8000000000000000ull);
}

// The greatest key of a warp's lanes and its lowest id, in every lane.
SLX_DEV void warp_best(uint64_t& key, int& id) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
  const bool a = (uint32_t)(key >> 32) == hi;
  const uint32_t lo = __reduce_max_sync(0xffffffffu, a ? (uint32_t)key : 0u);
  id = (int)__reduce_min_sync(0xffffffffu,
                              a && (uint32_t)key == lo ? (uint32_t)id : 0x7fffffffu);
  key = (uint64_t)hi << 32 | lo;
}

// A cluster of 8 CTAs per row; runs of 32 vectors of eight ids (a warp's
// load) go round the CTAs, because the ids that rules touch crowd at the
// vocabulary's start and the cluster waits for its slowest CTA.  Every thread
// requests its history entries, the logits (16-byte loads, all in flight
// together, before the mask's words are there) and the mask's words, and while
// they come the CTA builds its ids' words: zero, history (each pass over it
// two loads ahead), biases.  The vectors are then copied (masked ids -inf) and
// the touched ids listed with their values; a second pass computes the list
// with whole warps, in fp64, so picks between neighbouring values do not
// depend on the rounding of an intermediate.  Bound for a batch by those
// phases, one behind the other in the two CTAs that an SM holds (the words'
// shared memory, 64 registers a thread): 38 % of the issue slots, DRAM at a
// quarter; 128 rows of 151936 with 8000 past tokens each and every rule: 51 us in
// bf16 in a graph (59 with an emptied L2), 76 in fp32, whose ids take two passes
// over the history.  Beside 52 us in a graph: a bitmap of touched ids with counts
// for those alone (a quarter of the shared memory, four CTAs of 256 threads),
// which goes over the history twice, 80; the history split over the cluster,
// counted by atomics into the other CTAs' shared memory, 69.  For one row by the
// chain history -> words -> copy -> list -> cluster reduction.
template <typename T>
__global__ void __cluster_dims__(kLogitCluster, 1, 1)
    __launch_bounds__(kLogitThreads, 2) k_logits(const LogitArgs a) {
  extern __shared__ __align__(16) uint32_t s_word[];
  __shared__ uint16_t s_list[kLogitList];
  __shared__ T s_val[kLogitList];
  __shared__ int s_n;
  __shared__ uint64_t s_key[kLogitThreads / 32], c_key[kLogitCluster];
  __shared__ int s_id[kLogitThreads / 32], c_id[kLogitCluster];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int row = blockIdx.x / kLogitCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  // CTA 0's shared memory is written by the others at the end: a CTA that
  // has passed the matching wait knows that CTA 0 runs
  cluster.barrier_arrive();
  pdl_wait_primary();
  const slx_logit_rules& R = a.r;
  const T* x_row = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.V;
  T* o_row = a.out ? reinterpret_cast<T*>(a.out) + (size_t)row * a.V : nullptr;
  const uint32_t* mask = R.mask ? R.mask + (size_t)row * R.mask_stride : nullptr;
  // vectors start at 16-byte boundaries of the row's logits: vector k holds
  // ids 8 k - lead .. + 7, the first and last perhaps not whole
  constexpr int AL = 16 / sizeof(T);
  const int lead = (int)((reinterpret_cast<uintptr_t>(x_row) / sizeof(T)) % AL);
  const bool same =
      ((reinterpret_cast<uintptr_t>(x_row) ^ reinterpret_cast<uintptr_t>(o_row)) & 15) == 0;
  const int n_vec = (int)(((long long)a.V + lead + 7) / 8);
  // this CTA's q-th vector; a thread's next one is `hop` vectors on
  auto vec_at = [&](int q) { return ((q >> 5) * kLogitCluster + rank) * 32 + (q & 31); };
  constexpr int hop = kLogitThreads * kLogitCluster;
  const int q_end = ((n_vec + 31) / 32 + kLogitCluster - 1 - rank) / kLogitCluster * 32;
  Pick best = {-INFINITY, 0x7fffffff};
  float plain = -INFINITY;   // best of the ids no rule touches
  int plain_i = 0x7fffffff, first = 0x7fffffff;  // its id; the lowest allowed id
  int n_hist = 0, n_prompt = 0, bias0 = 0, bias1 = 0;
  const int32_t* hist = R.history + (size_t)row * R.history_stride;
  // entries up to a 16-byte boundary, then four at a time, the first ones
  // requested before their count is known
  int h0 = 0;
  constexpr int kAhead = 2;
  int4 ahead[kAhead];
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (R.history) {
    h0 = (int)((16 - (reinterpret_cast<uintptr_t>(hist) & 15)) / 4 % 4);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int e = h0 + 4 * (tid + i * kLogitThreads);
      if (e < R.history_stride - 3) ahead[i] = *reinterpret_cast<const int4*>(hist + e);
    }
    n_hist = R.n_history[row];
    n_prompt = R.n_prompt ? R.n_prompt[row] : 0;
    if (R.repetition) rep = R.repetition[row];
    if (R.frequency) freq = R.frequency[row];
    if (R.presence) pres = R.presence[row];
  }
  if (R.bias_ids) {
    bias0 = R.bias_start[row];
    bias1 = R.bias_start[row + 1];
  }
  constexpr int KV = kLogitVecs<T>;
  for (int q0 = 0; q0 < q_end; q0 += KV * kLogitThreads) {
    const int kb = vec_at(q0 + tid), idb = 8 * kb - lead;
    auto whole = [&](int id) { return id >= 0 && id <= a.V - 8; };
    Raw8<T> raw[KV];
    uint32_t ok[KV];  // allowed bits of each vector (ids outside the row are not)
#pragma unroll
    for (int v = 0; v < KV; ++v) {
      const int id = idb + v * hop * 8;
      ok[v] = kb + v * hop < n_vec ? 0xffu : 0u;
      if (!ok[v]) continue;
      if (whole(id)) {
        raw[v].load(x_row + id);
      } else {
        if (id < 0) ok[v] &= 0xffu << -id;
        if (id > a.V - 8) ok[v] &= 0xffu >> (id + 8 - a.V);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (ok[v] >> j & 1) raw[v].load1(j, x_row + id + j);
      }
    }
    if (mask) {
#pragma unroll
      for (int v = 0; v < KV; ++v) {
        if (!ok[v]) continue;
        // (hop * 8 is a multiple of 32: the same shift for every vector)
        const int id = idb + v * hop * 8;
        const int i0 = max(id, 0) >> 5, i1 = min(id + 7, a.V - 1) >> 5;
        const uint32_t w0 = mask[i0];
        if (lead == 0)
          ok[v] &= w0 >> (idb & 31);
        else
          ok[v] &= id < 0 ? w0 << -id : __funnelshift_r(w0, mask[i1], idb & 31);
      }
    }
    if (R.history || R.bias_ids) {
      const int n_id = min(q_end - q0, KV * kLogitThreads) * 8;
      if (q0 > 0) __syncthreads();
      for (int i = tid; i < n_id / 4; i += kLogitThreads)
        reinterpret_cast<uint4*>(s_word)[i] = make_uint4(0, 0, 0, 0);
      if (tid == 0) s_n = 0;
    }
    if (q0 == 0) {
      bool bad = n_hist < 0 || n_hist > R.history_stride || n_prompt < 0 || n_prompt > n_hist;
      n_hist = min(max(n_hist, 0), R.history_stride);
      n_prompt = min(max(n_prompt, 0), n_hist);
      bad = bad && R.history;
      if (R.bias_ids) {
        bad |= bias0 < 0 || bias1 < bias0 || bias1 > R.n_bias || bias1 - bias0 > kMaxBias;
        bias0 = min(max(bias0, 0), R.n_bias);
        bias1 = min(max(bias1, bias0), R.n_bias);
        bias1 = min(bias1, bias0 + kMaxBias);
      }
      if (bad && rank == 0 && tid == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      if (!R.history) n_hist = n_prompt = 0;
      h0 = min(h0, n_hist);
    }
    const bool words = n_hist > 0 || bias1 > bias0;
    if (words) {
      const int n_id = min(q_end - q0, KV * kLogitThreads) * 8;
      // place of an id's word in this pass, n_id or more if it is not here
      const unsigned base = (unsigned)q0 * 8;
      auto place = [&](int id) -> unsigned {
        const unsigned e = (unsigned)id + lead, run = e >> 8;
        return (unsigned)id < (unsigned)a.V && run % kLogitCluster == (unsigned)rank
                   ? (run / kLogitCluster << 8 | (e & 255u)) - base : 0xffffffffu;
      };
      const int b_first = bias0 + tid < bias1 ? R.bias_ids[bias0 + tid] : -1;
      __syncthreads();
      auto note = [&](int id, int e) {
        const unsigned at = place(id);
        if (at >= (unsigned)n_id) return;
        if (e >= n_prompt)
          atomicAdd(s_word + at, 1u);
        else if (!(reinterpret_cast<volatile uint32_t*>(s_word)[at] & kPrompt))
          atomicOr(s_word + at, kPrompt);
      };
      if (tid < h0) note(hist[tid], tid);
      auto note4 = [&](const int4& q, int e) {
        note(q.x, e);
        note(q.y, e + 1);
        note(q.z, e + 2);
        note(q.w, e + 3);
      };
      if (q0 > 0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int e = h0 + 4 * (tid + i * kLogitThreads);
          if (e < n_hist - 3) ahead[i] = *reinterpret_cast<const int4*>(hist + e);
        }
      }
#pragma unroll 1
      for (int e = h0 + 4 * tid;; e += 4 * kAhead * kLogitThreads) {
        int4 now[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          now[i] = ahead[i];
          const int en = e + 4 * (kAhead + i) * kLogitThreads;
          if (en < n_hist - 3) ahead[i] = *reinterpret_cast<const int4*>(hist + en);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (e + 4 * i * kLogitThreads < n_hist - 3) note4(now[i], e + 4 * i * kLogitThreads);
        if (e + 4 * kAhead * kLogitThreads >= n_hist - 3) break;
      }
      const int h1 = h0 + (n_hist - h0) / 4 * 4 + tid;
      if (h1 < n_hist) note(hist[h1], h1);
      // the row's last entry of an id stands
      auto bias = [&](int id, int e) {
        const unsigned at = place(id);
        if (at >= (unsigned)n_id) return;
        const uint32_t field = (uint32_t)(e - bias0 + 1) << kBiasShift;
        uint32_t old = reinterpret_cast<volatile uint32_t*>(s_word)[at];
        while ((old & ~kPrompt) >> kBiasShift < (uint32_t)(e - bias0 + 1)) {
          const uint32_t w = (old & (kPrompt | kCountMask)) | field;
          const uint32_t was = atomicCAS(s_word + at, old, w);
          if (was == old) break;
          old = was;
        }
      };
      bias(b_first, bias0 + tid);
      for (int e = bias0 + tid + kLogitThreads; e < bias1; e += kLogitThreads)
        bias(R.bias_ids[e], e);
      __syncthreads();
    }
    float pass = -INFINITY;  // best of this pass's ids that no rule touches,
    uint32_t pass_free = 0;  // its vector and the vector's such ids
    int pass_v = -1;
#pragma unroll
    for (int v = 0; v < KV; ++v) {
      const int q = v * kLogitThreads + tid, id = idb + v * hop * 8;
      uint32_t touched = 0;
      if (words && ok[v]) {
        const uint4 lo = reinterpret_cast<const uint4*>(s_word)[2 * q];
        const uint4 hi = reinterpret_cast<const uint4*>(s_word)[2 * q + 1];
        if (lo.x | lo.y | lo.z | lo.w | hi.x | hi.y | hi.z | hi.w)
          touched = (lo.x != 0) | (lo.y != 0) << 1 | (lo.z != 0) << 2 | (lo.w != 0) << 3 |
                    (hi.x != 0) << 4 | (hi.y != 0) << 5 | (hi.z != 0) << 6 | (hi.w != 0) << 7;
      }
      if (uint32_t list = touched & ok[v]) {
        int at = atomicAdd(&s_n, __popc(list));
        for (; list; list &= list - 1, ++at) {
          const int j = __ffs(list) - 1;
          if (at < kLogitList) {
            s_list[at] = (uint16_t)(q * 8 + j);
            s_val[at] = raw[v].bits(j);
          }
        }
      }
      if (ok[v]) first = min(first, id + __ffs(ok[v]) - 1);
      if (ok[v] != 0xffu) raw[v].mask(ok[v]);
      const uint32_t free = ok[v] & ~touched;  // ids no rule touches
      if (free) {
        float top;
        if (touched) {
          Raw8<T> r = raw[v];
          r.mask(free);
          top = r.top();
        } else {
          top = raw[v].top();
        }
        if (top > pass) {
          pass = top;
          pass_v = v;
          pass_free = free;
        }
      }
      if (o_row && kb + v * hop < n_vec) {
        if (whole(id) && same) {
          raw[v].store(o_row + id);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (id + j >= 0 && id + j < a.V) raw[v].store1(j, o_row + id + j);
        }
      }
    }
    if (pass > plain) {
      Raw8<T> r;
#pragma unroll
      for (int v = 0; v < KV; ++v)
        if (v == pass_v) r = raw[v];
      uint32_t at = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) at |= (uint32_t)(r.get(j) == pass) << j;
      plain = pass;
      plain_i = idb + pass_v * hop * 8 + __ffs(at & pass_free) - 1;
    }
    if (words) {
      const int n_id = min(q_end - q0, KV * kLogitThreads) * 8;
      __syncthreads();  // the copied vectors are written (out may be logits)
      const bool listed = s_n <= kLogitList;
      const int n = listed ? s_n : n_id;
#pragma unroll 1
      for (int t = tid; t < n; t += kLogitThreads) {
        const int i = listed ? s_list[t] : t;
        const uint32_t w = s_word[i];
        const int id = 8 * vec_at(q0 + (i >> 3)) - lead + (i & 7);
        if (!listed && (!w || (mask && !(mask[id >> 5] >> (id & 31) & 1u)))) continue;
        double x = to_f32(listed ? s_val[t] : x_row[id]);
        const uint32_t c = w & kCountMask;
        if (c || (w & kPrompt)) x = x > 0.0 ? x / (double)rep : x * (double)rep;
        if (c) x = __dsub_rn(__dsub_rn(x, __dmul_rn((double)freq, (double)c)), (double)pres);
        const int e = (int)((w & ~kPrompt) >> kBiasShift);
        if (e) x = __dadd_rn(x, (double)R.bias_values[bias0 + e - 1]);
        best.take(x, id);
        if (o_row) from_f32(o_row + id, (float)x);
      }
    }
  }
  cluster.barrier_wait();
  if (!a.pick) return;
  // an allowed id whose logit is -inf (or NaN) is picked only if all are
  if (first != 0x7fffffff) best.take(-INFINITY, first);
  if (plain_i != 0x7fffffff) best.take((double)plain, plain_i);
  // (key 0 is below every value's)
  uint64_t key = best.i == 0x7fffffff ? 0 : pick_key(best.v);
  int id = best.i;
  warp_best(key, id);
  if (lane == 0) {
    s_key[warp] = key;
    s_id[warp] = id;
  }
  __syncthreads();
  if (warp == 0) {
    constexpr int W = kLogitThreads / 32;
    key = s_key[lane % W];
    id = s_id[lane % W];
    warp_best(key, id);
    if (lane == 0) {
      *cluster.map_shared_rank(&c_key[rank], 0) = key;
      *cluster.map_shared_rank(&c_id[rank], 0) = id;
    }
  }
  cluster.sync();
  if (rank == 0 && warp == 0) {
    key = c_key[lane % kLogitCluster];
    id = c_id[lane % kLogitCluster];
    warp_best(key, id);
    if (lane == 0) a.pick[row] = id < a.V ? id : -1;
  }
}

int launch_logits(const LogitArgs& a, bool f32, cudaStream_t s) {
  static PerDevice configured;
  std::atomic<int>& slot = configured.here();
  if (!slot.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(k_logits<uint16_t>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kLogitSpan<uint16_t> * 4) != cudaSuccess ||
        cudaFuncSetAttribute(k_logits<float>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kLogitSpan<float> * 4) != cudaSuccess)
      return SLX_ERR_CUDA;
    slot.store(1, std::memory_order_relaxed);
  }
  if (a.T > 0x7fffffff / kLogitCluster || a.V > 0x7fffffff - 64) return SLX_ERR_UNSUPPORTED;
  // words of the ids a CTA handles in one pass: runs of 256, at most one more
  // than the alignment of a row's start allows for
  const long long runs = ((a.V + 7LL + 7) / 8 + 31) / 32;
  const long long ids = (runs + kLogitCluster - 1) / kLogitCluster * 256;
  const int span = f32 ? kLogitSpan<float> : kLogitSpan<uint16_t>;
  const bool words = a.r.history || a.r.bias_ids;
  const size_t smem = words ? (size_t)(ids < span ? ids : span) * 4 : 0;
  const dim3 grid((unsigned)a.T * kLogitCluster);
  const cudaError_t e =
      f32 ? launch_k(k_logits<float>, grid, dim3(kLogitThreads), smem, s, a)
          : launch_k(k_logits<uint16_t>, grid, dim3(kLogitThreads), smem, s, a);
  return e == cudaSuccess ? SLX_OK : SLX_ERR_CUDA;
}

}  // namespace slx
