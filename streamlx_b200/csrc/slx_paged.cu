// Batched decode over a paged key-value cache (sm_100a): the step's plan
// (block tables and slot maps from request lengths), q/k RMSNorm + RoPE +
// append to the pages, and attention of the new tokens over the pages.
// Page layout: [n_pages][2 (K, V)][n_kv][page_size][head_dim], so the keys of
// one kv head in one page are one contiguous block.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include "slx_kernels.cuh"

namespace slx {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ plan --

constexpr int kPlanThreads = 512;

// Largest i with s[i] <= v (s ascending, s[0] = 0 <= v < s[n]): the request
// an item belongs to, requests without items being skipped.
SLX_DEV int owner_of(const int32_t* s, int n, int v) {
  int lo = 0, hi = n;  // s[lo] <= v < s[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// Three prefix sums over the requests (rows, pages popped, pages pushed),
// then every pushed page, popped page and row finds its request by binary
// search.  One cluster: each CTA forms the sums itself, so the only things
// that cross CTAs are the state that is overwritten (read before the first
// cluster barrier, written after it) and the free stack (pushed before the
// second, popped after it).  Bound by its chain of dependent reads.
__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(const PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* s_row = plan_smem;               // [n_req + 1]
  int32_t* s_get = s_row + a.n_req + 1;     // [n_req + 1]
  int32_t* s_back = s_get + a.n_req + 1;    // [n_req + 1]
  int32_t* s_len = s_back + a.n_req + 1;    // [n_req]
  __shared__ long long w_sum[3][kPlanThreads / 32];
  __shared__ int s_bad;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int sh = 31 - __clz(a.page_size);
  const long long cap = (long long)a.max_pages << sh;
  pdl_launch_dependents();
  pdl_wait_primary();
  if (tid == 0) s_bad = 0;
  __syncthreads();
  const int per = (a.n_req + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
  auto pages = [&](long long n) { return (n + a.page_size - 1) >> sh; };
  // counts of request i; false when its numbers are out of range
  auto counts = [&](int i, long long (&c)[3], int& len) {
    const int nw = a.n_new[i];
    len = a.lengths[i];
    c[0] = c[1] = c[2] = 0;
    if (nw < -1 || len < 0 || len + (long long)max(nw, 0) > cap) return false;
    if (nw < 0) {
      c[2] = pages(len);
    } else {
      c[0] = nw;
      c[1] = pages((long long)len + nw) - pages(len);
    }
    return true;
  };
  long long sum[3] = {0, 0, 0};
  for (int i = r0; i < r1; ++i) {
    long long c[3];
    int len;
    if (!counts(i, c, len)) s_bad = 1;
    s_len[i] = len;
#pragma unroll
    for (int q = 0; q < 3; ++q) sum[q] += c[q];
  }
  long long inc[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    long long v = sum[q];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    inc[q] = v;
    if (lane == 31) w_sum[q][warp] = v;
  }
  const int n_free = *a.n_free;
  __syncthreads();
  long long tot[3], at[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    long long before = 0, all = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) before += w_sum[q][w];
      all += w_sum[q][w];
    }
    tot[q] = all;
    at[q] = before + inc[q] - sum[q];
  }
  int code = SLX_OK;
  if (s_bad || n_free < 0 || n_free + tot[2] > a.n_pages)
    code = SLX_ERR_OUT_OF_RANGE;
  else if (tot[0] > a.n_rows || tot[1] > n_free + tot[2])
    code = SLX_ERR_PAGES;
  if (code == SLX_OK) {
    for (int i = r0; i < r1; ++i) {
      long long c[3];
      int len;
      counts(i, c, len);
      s_row[i] = (int)at[0];
      s_get[i] = (int)at[1];
      s_back[i] = (int)at[2];
#pragma unroll
      for (int q = 0; q < 3; ++q) at[q] += c[q];
    }
    if (tid == 0) {
      s_row[a.n_req] = (int)tot[0];
      s_get[a.n_req] = (int)tot[1];
      s_back[a.n_req] = (int)tot[2];
    }
  }
  cluster.sync();  // every CTA has read lengths and n_free
  const int gt = cluster.block_rank() * kPlanThreads + tid;
  const int gn = cluster.num_blocks() * kPlanThreads;
  if (code != SLX_OK) {
    if (gt == 0) {
      set_status(a.status, code);
      *a.n_free_out = n_free;
    }
    for (int i = gt; i <= a.n_req; i += gn) {
      if (i < a.n_req) a.lengths_out[i] = s_len[i];
      a.row_start[i] = 0;
    }
    for (int r = gt; r < a.n_rows; r += gn)
      a.row_req[r] = a.row_pos[r] = a.row_slot[r] = -1;
    return;
  }
  const int n_back = (int)tot[2], n_get = (int)tot[1], n_rows = (int)tot[0];
  const int top = n_free + n_back;
  for (int g = gt; g < n_back; g += gn) {
    const int i = owner_of(s_back, a.n_req, g);
    a.free_list[n_free + g] = a.table[(size_t)i * a.max_pages + (g - s_back[i])];
  }
  for (int i = gt; i <= a.n_req; i += gn) {
    a.row_start[i] = s_row[i];
    if (i < a.n_req)
      a.lengths_out[i] = s_back[i + 1] > s_back[i] ? 0 : s_len[i] + s_row[i + 1] - s_row[i];
  }
  if (gt == 0) *a.n_free_out = top - n_get;
  cluster.sync();  // the pushed pages are on the stack
  // the page that is the g-th to be popped
  auto popped = [&](int g) {
    const int p = __ldcg(a.free_list + (top - 1 - g));
    if (p < 0 || p >= a.n_pages) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    return p;
  };
  for (int g = gt; g < n_get; g += gn) {
    const int i = owner_of(s_get, a.n_req, g);
    const int had = (int)pages(s_len[i]);
    a.table[(size_t)i * a.max_pages + had + (g - s_get[i])] = popped(g);
  }
  for (int r = gt; r < a.n_rows; r += gn) {
    int req = -1, pos = -1, slot = -1;
    if (r < n_rows) {
      req = owner_of(s_row, a.n_req, r);
      pos = s_len[req] + (r - s_row[req]);
      const int col = pos >> sh, had = (int)pages(s_len[req]);
      const int p = col < had ? a.table[(size_t)req * a.max_pages + col]
                              : popped(s_get[req] + (col - had));
      if (p < 0 || p >= a.n_pages)
        set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      else
        slot = (p << sh) + (pos & (a.page_size - 1));
    }
    a.row_req[r] = req;
    a.row_pos[r] = pos;
    a.row_slot[r] = slot;
  }
}

int launch_paged_plan(const PlanArgs& a, cudaStream_t s) {
  const size_t smem = (size_t)(4 * a.n_req + 3) * 4;
  static PerDevice configured;
  std::atomic<int>& slot = configured.here();
  if (!slot.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(k_paged_plan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (4 * 8192 + 3) * 4) != cudaSuccess)
      return SLX_ERR_CUDA;
    slot.store(1, std::memory_order_relaxed);
  }
  return launch_k(k_paged_plan, dim3(1), dim3(kPlanThreads), smem, s, a) ==
                 cudaSuccess ? SLX_OK : SLX_ERR_CUDA;
}

// ---------------------------------------------------------------- append --

SLX_DEV uint8_t f32_to_e4m3(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// One CTA per row.  The row's hd / 2 rotations once in shared memory (angle
// in fp64, reduced to one turn, then fp32 sine and cosine), then hd / 8
// lanes per head, eight elements each: the other half of a rotated pair sits
// hd / 16 lanes away.
constexpr int kAppendThreads = 256;

template <int HD, bool E4M3>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(const AppendArgs a) {
  constexpr int L = HD / 8;  // lanes per head
  __shared__ float s_cos[HD / 2], s_sin[HD / 2];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int t = blockIdx.x, nkv = a.kv.n_kv;
  const int p = a.pos[t];
  int slot = p < 0 ? -1 : a.slot[t];
  if (slot >= a.kv.n_pages * a.kv.page_size) {
    if (threadIdx.x == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    slot = -1;
  }
  if (slot < 0) {
    uint4* q = reinterpret_cast<uint4*>(a.q_out + (size_t)t * a.nq * HD);
    for (int i = threadIdx.x; i < a.nq * L; i += kAppendThreads)
      q[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x < HD / 2) {
    const double turn = 6.283185307179586476925286766559;
    double ang = (double)p * (double)a.inv_freq[threadIdx.x];
    ang -= rint(ang * (1.0 / turn)) * turn;
    float sn, cs;
    sincosf((float)ang, &sn, &cs);
    s_cos[threadIdx.x] = cs;
    s_sin[threadIdx.x] = sn;
  }
  __syncthreads();
  const int l = threadIdx.x % L;
  const uint16_t* row = a.qkv + (size_t)t * a.stride;
  const size_t ps = a.kv.page_size;
  const int page = slot / (int)ps, off = slot % (int)ps;
  const int heads = a.nq + 2 * nkv;
  // whole warps loop together (the head sums use shuffles)
  for (int h0 = 0; h0 < heads; h0 += kAppendThreads / L) {
    const int h = h0 + threadIdx.x / L;
    const bool on = h < heads;
    const uint4 raw = on ? reinterpret_cast<const uint4*>(row + (size_t)h * HD)[l]
                         : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = bf16_lo(w[q]);
      x[2 * q + 1] = bf16_hi(w[q]);
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const bool is_v = h >= a.nq + nkv;
    const uint16_t* nw = h < a.nq ? a.qn : a.kn;
    const float inv = rsqrtf(ss / (float)HD + a.eps);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float n = is_v ? x[j] : x[j] * inv * bf16_to_f32(nw[l * 8 + j]);
      const float other = __shfl_xor_sync(0xffffffffu, n, L / 2);
      const int i = (l % (L / 2)) * 8 + j;
      const float cs = s_cos[i], sn = s_sin[i];
      // first half a cos - b sin, second half b cos + a sin
      y[j] = is_v ? n : l < L / 2 ? n * cs - other * sn : n * cs + other * sn;
    }
    if (!on) continue;
    if (h < a.nq) {
      uint4 o;
      o.x = pack_bf16x2(y[0], y[1]);
      o.y = pack_bf16x2(y[2], y[3]);
      o.z = pack_bf16x2(y[4], y[5]);
      o.w = pack_bf16x2(y[6], y[7]);
      reinterpret_cast<uint4*>(a.q_out + ((size_t)t * a.nq + h) * HD)[l] = o;
      continue;
    }
    const int kh = is_v ? h - a.nq - nkv : h - a.nq;
    const size_t at = ((((size_t)page * 2 + is_v) * nkv + kh) * ps + off) * HD + l * 8;
    if (E4M3) {
      const float sc = is_v ? a.kv.v_scale[kh] : a.kv.k_scale[kh];
      uint32_t o[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o[j / 4] |= (uint32_t)f32_to_e4m3(y[j] / sc) << (8 * (j % 4));
      *reinterpret_cast<uint2*>(a.kv.base + at) = make_uint2(o[0], o[1]);
    } else {
      uint4 o;
      o.x = pack_bf16x2(y[0], y[1]);
      o.y = pack_bf16x2(y[2], y[3]);
      o.z = pack_bf16x2(y[4], y[5]);
      o.w = pack_bf16x2(y[6], y[7]);
      *reinterpret_cast<uint4*>(a.kv.base + 2 * at) = o;
    }
  }
}

int launch_paged_append(const AppendArgs& a, bool e4m3, cudaStream_t s) {
  auto k = a.kv.hd == 128 ? (e4m3 ? k_paged_append<128, true> : k_paged_append<128, false>)
                          : (e4m3 ? k_paged_append<64, true> : k_paged_append<64, false>);
  return launch_k(k, dim3(a.T), dim3(kAppendThreads), 0, s, a) == cudaSuccess
             ? SLX_OK : SLX_ERR_CUDA;
}

// ------------------------------------------------------------- attention --
//
// out[t, h] = sum_j softmax_j(scale q[t, h] . k_j) v_j.  Per kv head the group
// of G q heads shares every key and value, so the bytes bound it: 2 G flops
// per bf16 element.  The products still go to the tensor cores (G = 8 at HBM
// speed would take most of the fp32 units' rate), as
//   S^T [16 keys x 8 heads] = K [16 x hd] q^T,   O^T [hd x 8] += V^T P^T
// with mma.m16n8k16: M is keys / dims, so no row is padding (tcgen05's
// smallest M of 64 or 128 heads would be).  The contraction index of an MMA
// may be permuted on both sides alike, and the fragments are chosen so that
// each is 16 contiguous bytes of a key: keys and values go from global memory
// to fragments without shared memory.  V pairs two keys per register (byte
// permutes); S^T's accumulators become P^T's operand by movmatrix.
//
// P is rounded to two 16-bit parts (hi + lo: 16 bits or more in all), so the
// only rounding of note is the output's.  E4m3 keys and values become fp16
// exactly; q becomes fp16 times a power of two per head that puts its largest
// element at 2^12 .. 2^13 (exact down to 2^-26 of it).
//
// Work is cut into units of 16 keys of one kv head; every CTA gets the same
// number of consecutive units of the list (row, kv head, unit), whatever the
// rows' lengths.  A (row, kv head) that one CTA covers is written directly,
// the others leave (max, sum, O) parts that k_paged_join adds in order.

constexpr int kPaWarps = 4;
constexpr int kPaThreads = 32 * kPaWarps;
constexpr int kPaUnit = 16;

struct PaWork {       // workspace of one call
  int4* desc;         // [n] split (row, kv head): first, last CTA, row, head
  float* o;           // [2 CTAs][G][hd] parts: 2 w + 1 a segment's first
  float2* ml;         // [2 CTAs][G] max (log2), sum
};

SLX_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

SLX_DEV uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
SLX_DEV uint2 ld_stream8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v2.u32 {%0,%1}, [%2];"
               : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <bool BF16>
SLX_DEV void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                      uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

SLX_DEV uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// two e4m3 bytes -> fp16 pair (exact; NaN stays NaN)
SLX_DEV uint32_t e4m3x2(uint32_t w) {
  uint32_t d;
  asm("{.reg .b16 t, u; mov.b32 {t, u}, %1; cvt.rn.f16x2.e4m3x2 %0, t;}"
      : "=r"(d) : "r"(w));
  return d;
}

// Keys row t attends: pos + 1, 0 for an idle row or one out of range.
SLX_DEV int row_keys(const PagedAttnArgs& a, int t) {
  const int p = a.pos[t];
  if (p < 0) return 0;
  const int r = a.req ? a.req[t] : t;
  if (r < 0 || r >= a.n_req || p / a.kv.page_size >= a.max_pages) return 0;
  return p + 1;
}

template <int HD, bool E4M3, int NT>
__global__ void __launch_bounds__(kPaThreads) k_paged_attn(const PagedAttnArgs a,
                                                           const PaWork ws) {
  constexpr int ES = E4M3 ? 1 : 2;       // bytes per element
  constexpr int KQ = HD * ES / 64;       // 16-byte pieces of a key per lane
  constexpr int KS = HD / 16;            // MMA steps of q . k
  constexpr int MT = HD / 16;            // 16-dim tiles of O^T
  constexpr int PAD = HD + 4;
  __shared__ long long s_pre[kPaThreads + 1];
  __shared__ long long w_sum[kPaWarps];
  __shared__ int s_chunk;
  __shared__ float s_m[kPaWarps][8 * NT], s_l[kPaWarps][8 * NT];
  __shared__ __align__(16) float s_o[kPaWarps][8 * NT][PAD];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int w = blockIdx.x, nw = gridDim.x;
  const int nkv = a.kv.n_kv, G = a.nq / nkv, ps = a.kv.page_size;
  const int sh = 31 - __clz(ps);
  const bool by_row = (long long)a.T * nkv <= nw;  // how desc is indexed
  pdl_launch_dependents();
  pdl_wait_primary();
  // units before each thread's block of rows
  const int chunk = (a.T + kPaThreads - 1) / kPaThreads;
  {
    long long n = 0;
    const int t1 = min((tid + 1) * chunk, a.T);
    for (int t = tid * chunk; t < t1; ++t)
      n += (row_keys(a, t) + kPaUnit - 1) / kPaUnit;
    long long v = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) w_sum[warp] = v;
    __syncthreads();
    for (int i = 0; i < warp; ++i) v += w_sum[i];
    s_pre[tid + 1] = v;
    if (tid == 0) s_pre[0] = 0;
  }
  // idle rows: zeros (and the status of those out of range)
  for (int t = w; t < a.T; t += nw) {
    if (row_keys(a, t) > 0) continue;
    if (a.pos[t] >= 0 && tid == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    uint4* o = reinterpret_cast<uint4*>(a.out + (size_t)t * a.nq * HD);
    for (int i = tid; i < a.nq * HD / 8; i += kPaThreads) o[i] = make_uint4(0, 0, 0, 0);
    if (by_row)
      for (int i = tid; i < nkv; i += kPaThreads) ws.desc[t * nkv + i] = make_int4(-1, 0, 0, 0);
  }
  __syncthreads();
  const long long total = s_pre[kPaThreads] * nkv;
  // units per CTA: a multiple of the warps (a step is one unit per warp)
  long long per = (total + nw - 1) / nw;
  per = (per + kPaWarps - 1) / kPaWarps * kPaWarps;
  if (per < kPaWarps) per = kPaWarps;
  long long x = w * per;
  const long long x_end = min(x + per, total);
  int4 my_desc = make_int4(-1, 0, 0, 0);
  if (x < x_end) {
    // the row unit x is in: its block of rows, then 32 rows at a time
    if (s_pre[tid] * nkv <= x && x < s_pre[tid + 1] * nkv) s_chunk = tid;
    __syncthreads();
    int rb = s_chunk * chunk;             // first row of the warp's 32
    long long before = s_pre[s_chunk] * nkv;
    int row = -1, keys, units, len_l;     // len_l: keys of row rb + lane
    for (;; rb += 32) {
      len_l = rb + lane < a.T ? row_keys(a, rb + lane) : 0;
      const int n = (len_l + kPaUnit - 1) / kPaUnit;
      long long v = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      const bool here = before + (v - n) * nkv <= x && x < before + v * nkv;
      const unsigned hit = __ballot_sync(0xffffffffu, here);
      if (hit) {
        const int i = __ffs(hit) - 1;
        row = rb + i;
        before += (__shfl_sync(0xffffffffu, v, i) - __shfl_sync(0xffffffffu, n, i)) * nkv;
        break;
      }
      before += __shfl_sync(0xffffffffu, v, 31) * nkv;
    }
    keys = __shfl_sync(0xffffffffu, len_l, row - rb);
    units = (keys + kPaUnit - 1) / kPaUnit;
    int kh = (int)((x - before) / units);
    int u0 = (int)((x - before) % units);
    while (true) {
      const int u1 = (int)min((long long)units, u0 + (x_end - x));
      const int req = a.req ? a.req[row] : row;
      const int32_t* tab = a.table + (size_t)req * a.max_pages;
      // q^T fragments of the group's heads
      uint32_t qf[NT][KS][2];
      float fac[NT][2];  // of heads 2c, 2c + 1: scores in log2 units
      const float fs = a.scale * 1.4426950408889634f * (E4M3 ? a.kv.k_scale[kh] : 1.f);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + g;
        const uint8_t* qp = reinterpret_cast<const uint8_t*>(
            a.q + (size_t)row * a.q_stride + (size_t)(kh * G + h) * HD);
        if constexpr (!E4M3) {
#pragma unroll
          for (int q = 0; q < KQ; ++q) {
            const uint4 v = h < G ? *reinterpret_cast<const uint4*>(qp + q * 64 + c * 16)
                                  : make_uint4(0, 0, 0, 0);
            qf[nt][2 * q][0] = v.x;
            qf[nt][2 * q][1] = v.y;
            qf[nt][2 * q + 1][0] = v.z;
            qf[nt][2 * q + 1][1] = v.w;
          }
          fac[nt][0] = fac[nt][1] = fs;
        } else {
          uint4 v[2 * KQ];
          float mx = 0.f;
#pragma unroll
          for (int q = 0; q < 2 * KQ; ++q) {
            v[q] = h < G ? *reinterpret_cast<const uint4*>(qp + (q >> 1) * 128 + c * 32 + (q & 1) * 16)
                         : make_uint4(0, 0, 0, 0);
            const uint32_t u[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(u[i])), fabsf(bf16_hi(u[i]))));
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // 2^k: the largest element lands in [2^12, 2^13)
          const int e = (int)(__float_as_uint(mx) >> 23) - 127;
          const int k = mx == 0.f || e == 128 ? 0 : min(12 - e, 100);
          const float up = __uint_as_float((uint32_t)(127 + k) << 23);
          const float down = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
          for (int q = 0; q < 2 * KQ; ++q) {
            const uint32_t u[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              qf[nt][2 * q + (i >> 1)][i & 1] = pack_f16x2(bf16_lo(u[i]) * up, bf16_hi(u[i]) * up);
          }
          // lane 8c holds head 2c's factor, lane 8c + 4 head 2c + 1's
          fac[nt][0] = fs * __shfl_sync(0xffffffffu, down, 8 * c);
          fac[nt][1] = fs * __shfl_sync(0xffffffffu, down, 8 * c + 4);
        }
      }
      float acc[NT][MT][4];
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
      }
      const size_t v_off = (size_t)nkv * ps * HD * ES;
      int u = u0 + warp;
      int page = u < u1 ? tab[(u * kPaUnit) >> sh] : 0;
      for (; u < u1; u += kPaWarps) {
        const int k0 = u * kPaUnit;
        const int next = u + kPaWarps < u1 ? tab[((u + kPaWarps) * kPaUnit) >> sh] : 0;
        if (page < 0 || page >= a.kv.n_pages) {
          if (lane == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
          page = next;
          continue;
        }
        const int last = min(kPaUnit, keys - k0) - 1;  // last key held
        const uint8_t* kp = a.kv.base +
            (((size_t)page * 2 * nkv + kh) * ps + (k0 & (ps - 1))) * (HD * ES);
        const uint8_t* vp = kp + v_off;
        page = next;
        uint4 kr[2][KQ];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t* p = kp + min(g + 8 * r, last) * (HD * ES) + c * 16;
#pragma unroll
          for (int q = 0; q < KQ; ++q) kr[r][q] = ld_stream(p + q * 64);
        }
        // value words of keys 2c, 2c + 1, 2c + 8, 2c + 9
        constexpr int VW = HD * ES / 32;  // words per lane and key
        uint32_t vr[4][VW];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = 2 * c + (r & 1) + 8 * (r >> 1);
          const uint8_t* p = vp + min(key, last) * (HD * ES) + g * (VW >= 4 ? 16 : 8);
          if constexpr (VW >= 4) {
#pragma unroll
            for (int q = 0; q < VW / 4; ++q) {
              const uint4 v = ld_stream(p + q * 128);
              vr[r][4 * q] = v.x;
              vr[r][4 * q + 1] = v.y;
              vr[r][4 * q + 2] = v.z;
              vr[r][4 * q + 3] = v.w;
            }
          } else {
            const uint2 v = ld_stream8(p);
            vr[r][0] = v.x;
            vr[r][1] = v.y;
          }
          if (last < kPaUnit - 1 && key > last) {
#pragma unroll
            for (int q = 0; q < VW; ++q) vr[r][q] = 0;
          }
        }
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int q = 0; q < KQ; ++q) {
          const uint32_t lo[4] = {kr[0][q].x, kr[0][q].y, kr[0][q].z, kr[0][q].w};
          const uint32_t hi[4] = {kr[1][q].x, kr[1][q].y, kr[1][q].z, kr[1][q].w};
          if constexpr (!E4M3) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<true>(s[nt], lo[2 * i], hi[2 * i], lo[2 * i + 1], hi[2 * i + 1],
                               qf[nt][2 * q + i][0], qf[nt][2 * q + i][1]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = e4m3x2(lo[i]), a2 = e4m3x2(lo[i] >> 16);
              const uint32_t a1 = e4m3x2(hi[i]), a3 = e4m3x2(hi[i] >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<false>(s[nt], a0, a1, a2, a3, qf[nt][4 * q + i][0],
                                qf[nt][4 * q + i][1]);
            }
          }
        }
        uint32_t ph[NT][2], pl[NT][2];  // P^T operands: hi and lo parts
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            p[i] = g + 8 * (i >> 1) <= last ? s[nt][i] * fac[nt][i & 1] : -INFINITY;
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = fmaxf(p[i], p[i + 2]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[nt][i]);
            const float ms = mx == -INFINITY ? 0.f : mx;
            f[i] = exp2_fast(m[nt][i] - ms);
            m[nt][i] = mx;
            p[i] = exp2_fast(p[i] - ms);
            p[i + 2] = exp2_fast(p[i + 2] - ms);
            l[nt][i] = l[nt][i] * f[i] + (p[i] + p[i + 2]);
          }
          if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              acc[nt][i][0] *= f[0];
              acc[nt][i][1] *= f[1];
              acc[nt][i][2] *= f[0];
              acc[nt][i][3] *= f[1];
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t hi, lo;
            if constexpr (!E4M3) {
              hi = pack_bf16x2(p[2 * i], p[2 * i + 1]);
              lo = pack_bf16x2(p[2 * i] - bf16_lo(hi), p[2 * i + 1] - bf16_hi(hi));
            } else {
              hi = pack_f16x2(p[2 * i], p[2 * i + 1]);
              const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              lo = pack_f16x2(p[2 * i] - b.x, p[2 * i + 1] - b.y);
            }
            ph[nt][i] = transpose8x8(hi);
            pl[nt][i] = transpose8x8(lo);
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t a0, a1, a2, a3;
          if constexpr (!E4M3) {
            // word i of the lane's dims: dims 2i (low halves) and 2i + 1
            a0 = __byte_perm(vr[0][i], vr[1][i], 0x5410);
            a1 = __byte_perm(vr[0][i], vr[1][i], 0x7632);
            a2 = __byte_perm(vr[2][i], vr[3][i], 0x5410);
            a3 = __byte_perm(vr[2][i], vr[3][i], 0x7632);
          } else {
            // bytes 2 (i % 2), + 1 of word i / 2: dims 2i and 2i + 1
            const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
            const uint32_t lo = __byte_perm(vr[0][i >> 1], vr[1][i >> 1], sel);
            const uint32_t hi = __byte_perm(vr[2][i >> 1], vr[3][i >> 1], sel);
            a0 = e4m3x2(lo);
            a1 = e4m3x2(lo >> 16);
            a2 = e4m3x2(hi);
            a3 = e4m3x2(hi >> 16);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<!E4M3>(acc[nt][i], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
            mma16816<!E4M3>(acc[nt][i], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
          }
        }
      }
      // the warps' states into shared memory: O in dim order per head
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = l[nt][i];
          v += __shfl_xor_sync(0xffffffffu, v, 4);
          v += __shfl_xor_sync(0xffffffffu, v, 8);
          v += __shfl_xor_sync(0xffffffffu, v, 16);
          const int h = nt * 8 + 2 * c + i;
          if (g == 0) {
            s_m[warp][h] = m[nt][i];
            s_l[warp][h] = v;
          }
#pragma unroll
          for (int j = 0; j < MT; j += 2) {
            // tiles j, j + 1: four consecutive dims
            const int d = E4M3 ? g * (HD / 8) + 2 * j : (j / 4) * 64 + g * 8 + (j % 4) * 2;
            *reinterpret_cast<float4*>(&s_o[warp][h][d]) = make_float4(
                acc[nt][j][i], acc[nt][j][i + 2], acc[nt][j + 1][i], acc[nt][j + 1][i + 2]);
          }
        }
      }
      __syncthreads();
      const bool whole = u0 == 0 && u1 == units;
      const int part = 2 * w + (u0 == 0 ? 1 : 0);
      const float sv = E4M3 ? a.kv.v_scale[kh] : 1.f;
      for (int i = tid; i < G * (HD / 4); i += kPaThreads) {
        const int h = i / (HD / 4), d = (i % (HD / 4)) * 4;
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < kPaWarps; ++k) M = fmaxf(M, s_m[k][h]);
        const float Mf = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kPaWarps; ++k) {
          const float f = exp2_fast(s_m[k][h] - Mf);
          const float4 v = *reinterpret_cast<const float4*>(&s_o[k][h][d]);
          L += f * s_l[k][h];
          o.x += f * v.x;
          o.y += f * v.y;
          o.z += f * v.z;
          o.w += f * v.w;
        }
        o.x *= sv;
        o.y *= sv;
        o.z *= sv;
        o.w *= sv;
        if (whole) {
          *reinterpret_cast<uint2*>(a.out + ((size_t)row * a.nq + kh * G + h) * HD + d) =
              make_uint2(pack_bf16x2(o.x / L, o.y / L), pack_bf16x2(o.z / L, o.w / L));
        } else {
          *reinterpret_cast<float4*>(ws.o + ((size_t)part * G + h) * HD + d) = o;
          if (d == 0) ws.ml[(size_t)part * G + h] = make_float2(M, L);
        }
      }
      if (u0 == 0) {
        const int4 d = whole ? make_int4(-1, 0, 0, 0)
                             : make_int4(w, (int)((x + units - 1) / per), row, kh);
        if (by_row) {
          if (tid == 0) ws.desc[row * nkv + kh] = d;
        } else if (!whole) {
          my_desc = d;
        }
      }
      x += u1 - u0;
      if (x >= x_end) break;
      __syncthreads();  // s_o is read before the next segment's is written
      u0 = 0;
      if (++kh == nkv) {
        kh = 0;
        // the next row with keys (there is one: x < total)
        unsigned more = __ballot_sync(0xffffffffu, len_l > 0 && rb + lane > row);
        while (!more) {
          rb += 32;
          len_l = rb + lane < a.T ? row_keys(a, rb + lane) : 0;
          more = __ballot_sync(0xffffffffu, len_l > 0);
        }
        row = rb + __ffs(more) - 1;
        keys = __shfl_sync(0xffffffffu, len_l, row - rb);
        units = (keys + kPaUnit - 1) / kPaUnit;
      }
    }
  }
  if (!by_row && tid == 0) ws.desc[w] = my_desc;
}

// Parts of one split (row, kv head), one q head per CTA: added in order of
// the keys, eight parts at a time per warp group.
constexpr int kJoinThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const PagedAttnArgs a,
                                                             const PaWork ws) {
  constexpr int TP = HD / 4;                 // threads per part
  constexpr int NG = kJoinThreads / TP;      // parts at a time
  __shared__ float s_red[kJoinThreads / 32];
  __shared__ float s_l[NG];
  __shared__ __align__(16) float s_o[NG][HD];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int4 d = ws.desc[blockIdx.x];
  if (d.x < 0) return;
  const int G = a.nq / a.kv.n_kv, h = blockIdx.y;
  const int n = d.y - d.x + 1;
  const int tid = threadIdx.x;
  // part i of the segment: the first CTA's second slot, then first slots
  auto part = [&](int i) { return (size_t)(2 * (d.x + i) + (i == 0 ? 1 : 0)) * G + h; };
  float M = -INFINITY;
  for (int i = tid; i < n; i += kJoinThreads) M = fmaxf(M, ws.ml[part(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_red[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) M = fmaxf(M, s_red[i]);
  if (M == -INFINITY) M = 0.f;
  const int q = tid / TP, d4 = (tid % TP) * 4;
  float L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = q; i < n; i += NG) {
    const size_t p = part(i);
    const float2 ml = ws.ml[p];
    const float4 v = *reinterpret_cast<const float4*>(ws.o + p * HD + d4);
    const float f = exp2_fast(ml.x - M);
    L += f * ml.y;
    o.x += f * v.x;
    o.y += f * v.y;
    o.z += f * v.z;
    o.w += f * v.w;
  }
  *reinterpret_cast<float4*>(&s_o[q][d4]) = o;
  if (d4 == 0) s_l[q] = L;
  __syncthreads();
  if (tid < HD) {
    float O = 0.f;
    L = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      O += s_o[i][tid];
      L += s_l[i];
    }
    a.out[((size_t)d.z * a.nq + d.w * G + h) * HD + tid] = f32_to_bf16(O / L);
  }
}

namespace {

using AttnKernel = void (*)(PagedAttnArgs, PaWork);

AttnKernel attn_kernel(int hd, bool e4m3, int G, int* id) {
  static const AttnKernel k[8] = {
      k_paged_attn<64, false, 1>,  k_paged_attn<64, false, 2>,
      k_paged_attn<64, true, 1>,   k_paged_attn<64, true, 2>,
      k_paged_attn<128, false, 1>, k_paged_attn<128, false, 2>,
      k_paged_attn<128, true, 1>,  k_paged_attn<128, true, 2>};
  *id = (hd == 128 ? 4 : 0) + (e4m3 ? 2 : 0) + (G > 8 ? 1 : 0);
  return k[*id];
}

constexpr int kPaMaxCtas = 1024;  // CTAs of a launch (workspace size)

// CTAs that fill the current device; 0 on a CUDA error.
int attn_ctas(AttnKernel k, int id) {
  static PerDevice known[8];
  std::atomic<int>& slot = known[id].here();
  int n = slot.load(std::memory_order_relaxed);
  if (!n) {
    int dev = 0, sms = 0, per_sm = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, kPaThreads, 0) != cudaSuccess)
      return 0;
    n = sms * per_sm < kPaMaxCtas ? sms * per_sm : kPaMaxCtas;
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace

// desc | parts' O | parts' (max, sum), for the largest launch
size_t paged_attn_workspace_bytes(int T, int nq, int nkv, int hd) {
  if (T == 0) return 0;
  const size_t G = nq / nkv;
  return kPaMaxCtas * (sizeof(int4) + 2 * G * (hd * sizeof(float) + sizeof(float2)));
}

int launch_paged_attn(const PagedAttnArgs& a, bool e4m3, cudaStream_t s) {
  const int nkv = a.kv.n_kv, G = a.nq / nkv;
  int id;
  const AttnKernel k = attn_kernel(a.kv.hd, e4m3, G, &id);
  const int full = attn_ctas(k, id);
  if (full < 1) return SLX_ERR_CUDA;
  // no more CTAs than steps (a unit per warp) the rows could fill
  const long long segs = (long long)a.T * nkv;
  int grid = full;
  if (segs < (long long)full * kPaWarps) {
    const long long row_units = (long long)a.max_pages * (a.kv.page_size / kPaUnit);
    const long long steps = (segs * row_units + kPaWarps - 1) / kPaWarps;
    if (steps < full) grid = (int)steps;
  }
  PaWork ws;
  uint8_t* p = reinterpret_cast<uint8_t*>(a.ws);
  ws.desc = reinterpret_cast<int4*>(p);
  ws.o = reinterpret_cast<float*>(p + kPaMaxCtas * sizeof(int4));
  ws.ml = reinterpret_cast<float2*>(ws.o + (size_t)kPaMaxCtas * 2 * G * a.kv.hd);
  if (launch_k(k, dim3(grid), dim3(kPaThreads), 0, s, a, ws) != cudaSuccess)
    return SLX_ERR_CUDA;
  const dim3 jgrid((unsigned)(segs <= grid ? segs : grid), G);
  auto j = a.kv.hd == 128 ? k_paged_join<128> : k_paged_join<64>;
  return launch_chained(j, jgrid, dim3(kJoinThreads), 0, s, a, ws) == cudaSuccess
             ? SLX_OK : SLX_ERR_CUDA;
}

}  // namespace slx
