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

size_t paged_attn_workspace_bytes(int T, int nq, int nkv, int hd) { return 0; }

// One CTA per (kv head, row), a warp per key: the simplest form.
template <int HD, bool E4M3>
__global__ void __launch_bounds__(128) k_paged_attn(const PagedAttnArgs a) {
  constexpr int D = HD / 32;  // dims per lane
  constexpr int kMaxG = 16;
  __shared__ float s_o[4][kMaxG][HD];
  __shared__ float s_m[4][kMaxG], s_l[4][kMaxG];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkv = a.kv.n_kv, G = a.nq / nkv, ps = a.kv.page_size;
  const int kh = blockIdx.x % nkv, t = blockIdx.x / nkv;
  int p = a.pos[t];
  const int req = a.req ? a.req[t] : t;
  if (p >= 0 && (req < 0 || req >= a.n_req || p / ps >= a.max_pages)) {
    if (threadIdx.x == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    p = -1;
  }
  float q[kMaxG][D], o[kMaxG][D], m[kMaxG], l[kMaxG];
  const float sk = E4M3 ? a.kv.k_scale[kh] : 1.f, sv = E4M3 ? a.kv.v_scale[kh] : 1.f;
#pragma unroll
  for (int g = 0; g < kMaxG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) {
      o[g][d] = 0.f;
      q[g][d] = g < G ? bf16_to_f32(a.q[(size_t)t * a.q_stride + (size_t)(kh * G + g) * HD + lane * D + d]) : 0.f;
    }
  }
  for (int j = warp; j <= p; j += 4) {
    const int page = a.table[(size_t)req * a.max_pages + j / ps];
    if (page < 0 || page >= a.kv.n_pages) {
      if (lane == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      continue;
    }
    const size_t at = (((size_t)page * 2 * nkv + kh) * ps + j % ps) * HD + lane * D;
    const size_t v_at = at + (size_t)nkv * ps * HD;
    float k[D], v[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (E4M3) {
        const __nv_fp8_storage_t kb = a.kv.base[at + d], vb = a.kv.base[v_at + d];
        k[d] = __half2float(__half(__nv_cvt_fp8_to_halfraw(kb, __NV_E4M3))) * sk;
        v[d] = __half2float(__half(__nv_cvt_fp8_to_halfraw(vb, __NV_E4M3))) * sv;
      } else {
        k[d] = bf16_to_f32(reinterpret_cast<const uint16_t*>(a.kv.base)[at + d]);
        v[d] = bf16_to_f32(reinterpret_cast<const uint16_t*>(a.kv.base)[v_at + d]);
      }
    }
#pragma unroll
    for (int g = 0; g < kMaxG; ++g) {
      if (g >= G) break;
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < D; ++d) s += q[g][d] * k[d];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= a.scale;
      const float mn = fmaxf(m[g], s);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float f = expf(m[g] - ms), e = expf(s - ms);
      l[g] = l[g] * f + e;
#pragma unroll
      for (int d = 0; d < D; ++d) o[g][d] = o[g][d] * f + e * v[d];
      m[g] = mn;
    }
  }
#pragma unroll
  for (int g = 0; g < kMaxG; ++g) {
    s_m[warp][g] = m[g];
    s_l[warp][g] = l[g];
#pragma unroll
    for (int d = 0; d < D; ++d) s_o[warp][g][lane * D + d] = o[g][d];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * HD; i += 128) {
    const int g = i / HD, d = i % HD;
    float M = -INFINITY, Ls = 0.f, O = 0.f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w][g]);
    if (M == -INFINITY) M = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = expf(s_m[w][g] - M);
      Ls += s_l[w][g] * f;
      O += s_o[w][g][d] * f;
    }
    a.out[((size_t)t * a.nq + kh * G + g) * HD + d] = f32_to_bf16(p < 0 ? 0.f : O / Ls);
  }
}

int launch_paged_attn(const PagedAttnArgs& a, bool e4m3, cudaStream_t s) {
  auto k = a.kv.hd == 128 ? (e4m3 ? k_paged_attn<128, true> : k_paged_attn<128, false>)
                          : (e4m3 ? k_paged_attn<64, true> : k_paged_attn<64, false>);
  if ((long long)a.T * a.kv.n_kv > 0x7fffffff) return SLX_ERR_UNSUPPORTED;
  return launch_k(k, dim3(a.kv.n_kv * a.T), dim3(128), 0, s, a) == cudaSuccess
             ? SLX_OK : SLX_ERR_CUDA;
}

}  // namespace slx
