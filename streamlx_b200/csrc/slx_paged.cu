// Batched decode over a paged key-value cache (sm_100a): the step's plan
// (block tables and slot maps from request lengths), q/k RMSNorm + RoPE +
// append to the pages, and attention of the new tokens over the pages.
// Page layout: [n_pages][2 (K, V)][n_kv][page_size][head_dim], so the keys of
// one kv head in one page are one contiguous block.
#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "slx_paged.cuh"

namespace slx {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ plan --

constexpr int kPlanThreads = 512;
constexpr int kPlanCluster = 8;

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
  __shared__ __align__(16) int w_sum[3][kPlanThreads / 32];
  __shared__ int s_bad;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int sh = 31 - __clz(a.page_size);
  const long long cap = (long long)a.max_pages << sh;
  pdl_launch_dependents();
  pdl_wait_primary();
  if (tid == 0) s_bad = 0;
  __syncthreads();
  const int n_free = *a.n_free;
  const int per = (a.n_req + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(tid * per, a.n_req), r1 = min(r0 + per, a.n_req);
  auto pages = [&](long long n) { return (int)((n + a.page_size - 1) >> sh); };
  // sums stop at 2^31 - 1: more rows or pages than any step can have
  auto add = [](int x, int y) { return (int)min((unsigned)x + (unsigned)y, 0x7fffffffu); };
  int sum[3] = {0, 0, 0};
  for (int i = r0; i < r1; ++i) {
    const int nw = a.n_new[i], len = a.lengths[i];
    int c[3] = {0, 0, 0};
    if (nw < -1 || len < 0 || len + (long long)max(nw, 0) > cap) {
      s_bad = 1;
    } else if (nw < 0) {
      c[2] = pages(len);
    } else {
      c[0] = nw;
      c[1] = pages((long long)len + nw) - pages(len);
    }
    s_len[i] = len;
    s_row[i] = c[0];
    s_get[i] = c[1];
    s_back[i] = c[2];
#pragma unroll
    for (int q = 0; q < 3; ++q) sum[q] = add(sum[q], c[q]);
  }
  int inc[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    int v = sum[q];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = add(v, u);
    }
    inc[q] = v;
    if (lane == 31) w_sum[q][warp] = v;
  }
  __syncthreads();
  int tot[3], at[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w == warp) before = all;
      all = add(all, w_sum[q][w]);
    }
    tot[q] = all;
    at[q] = add(before, inc[q]) - sum[q];
  }
  int code = SLX_OK;
  if (s_bad || n_free < 0 || n_free > a.n_pages || tot[2] > a.n_pages - n_free)
    code = SLX_ERR_OUT_OF_RANGE;
  else if (tot[0] > a.n_rows || tot[1] > n_free + tot[2])
    code = SLX_ERR_PAGES;
  if (code == SLX_OK) {
    for (int i = r0; i < r1; ++i) {
      int32_t* const pre[3] = {s_row, s_get, s_back};
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        const int c = pre[q][i];
        pre[q][i] = at[q];
        at[q] += c;
      }
    }
    if (tid == 0) {
      s_row[a.n_req] = tot[0];
      s_get[a.n_req] = tot[1];
      s_back[a.n_req] = tot[2];
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
  const int n_back = tot[2], n_get = tot[1], n_rows = tot[0];
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
  // four items at a time: their reads of the stack and the table overlap
  constexpr int B = 4;
  for (int g0 = gt; g0 < n_get; g0 += B * gn) {
    int p[B];
#pragma unroll
    for (int j = 0; j < B; ++j)
      p[j] = g0 + j * gn < n_get ? __ldcg(a.free_list + (top - 1 - (g0 + j * gn))) : 0;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int g = g0 + j * gn;
      if (g >= n_get) break;
      const int i = owner_of(s_get, a.n_req, g);
      if (p[j] < 0 || p[j] >= a.n_pages) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      a.table[(size_t)i * a.max_pages + pages(s_len[i]) + (g - s_get[i])] = p[j];
    }
  }
  for (int t0 = gt; t0 < a.n_rows; t0 += B * gn) {
    int req[B], pos[B], p[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int r = t0 + j * gn;
      req[j] = pos[j] = p[j] = -1;
      if (r < n_rows) {
        const int i = owner_of(s_row, a.n_req, r);
        req[j] = i;
        pos[j] = s_len[i] + (r - s_row[i]);
        const int col = pos[j] >> sh, had = pages(s_len[i]);
        // an old page from the table, a new one as it was popped
        p[j] = col < had ? a.table[(size_t)i * a.max_pages + col]
                         : __ldcg(a.free_list + (top - 1 - (s_get[i] + (col - had))));
      }
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int r = t0 + j * gn;
      if (r >= a.n_rows) break;
      int slot = -1;
      if (p[j] >= 0 && p[j] < a.n_pages)
        slot = (p[j] << sh) + (pos[j] & (a.page_size - 1));
      else if (r < n_rows)
        set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      a.row_req[r] = req[j];
      a.row_pos[r] = pos[j];
      a.row_slot[r] = slot;
    }
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
  // one CTA while each of its threads has a few rows at most (the cluster's
  // barriers cost about 1 us), else a cluster of eight
  if (a.n_rows + a.n_req <= 4 * kPlanThreads)
    return launch_k(k_paged_plan, dim3(1), dim3(kPlanThreads), smem, s, a) ==
                   cudaSuccess ? SLX_OK : SLX_ERR_CUDA;
  return launch_cluster(kPlanCluster, k_paged_plan, dim3(kPlanCluster), dim3(kPlanThreads),
                        smem, s, a) == cudaSuccess ? SLX_OK : SLX_ERR_CUDA;
}

// ---------------------------------------------------------------- append --

// four values to e4m3, to nearest, saturating at 448
SLX_DEV uint32_t f32x4_to_e4m3(const float (&x)[4]) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// One CTA per row, hd / 8 lanes per head, each with four elements of the
// head's first half and the four they are rotated with.  The row's heads are
// requested first; while they come, hd / 2 threads form the row's rotations
// (the angle in turns, in fp64, less its whole turns).  Keys of e4m3 pages go
// through fp64 up to their one rounding: with a step of 2^-3, a value that
// fp32 leaves on the wrong side of a step's middle would be off by far more
// than fp32's own error.  Bound by each row's chain position -> rotations ->
// barrier -> stores; of many rows 37 % of an SM's warps are there to cover it (64
// registers a thread), and 47 % of the issue slots are taken: 4096 rows, 16/2
// heads of 128, in a graph: 15.2 us in e4m3, 10.6 in bf16 (6.1 and 6.4 us of
// bytes).
constexpr int kAppendThreads = 128;
constexpr int kAppendAhead = 4;  // passes over the heads requested together

// Four elements of each half of a head (bf16).
struct HalfPair {
  uint2 a, b;
  template <typename R>
  SLX_DEV void get(R (&x)[4], R (&y)[4]) const {
    x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x); x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
    y[0] = bf16_lo(b.x); y[1] = bf16_hi(b.x); y[2] = bf16_lo(b.y); y[3] = bf16_hi(b.y);
  }
};

template <int HD, bool E4M3>
__global__ void __launch_bounds__(kAppendThreads, 8) k_paged_append(const AppendArgs a) {
  constexpr int L = HD / 8;                // lanes per head
  constexpr int PH = kAppendThreads / L;   // heads per pass
  __shared__ __align__(16) float2 s_rot[HD / 2];  // cosine, sine
  __shared__ __align__(16) double2 s_rot_k[E4M3 ? HD / 2 : 1];  // the keys', where they are fp64
  pdl_launch_dependents();
  const int l = threadIdx.x % L, lh = threadIdx.x / L;
  auto load = [&](const uint16_t* head) {
    return HalfPair{reinterpret_cast<const uint2*>(head)[l],
                    reinterpret_cast<const uint2*>(head + HD / 2)[l]};
  };
  // fixed inputs, before the wait
  const HalfPair wq = load(a.qn), wk = load(a.kn);
  const double freq = threadIdx.x < HD / 2 ? (double)a.inv_freq[threadIdx.x] : 0.0;
  pdl_wait_primary();
  const int t = blockIdx.x, nkv = a.kv.n_kv;
  const uint16_t* row = a.qkv + (size_t)t * a.stride;
  const int p = a.pos[t];
  int slot = a.slot[t];
  // the first pass over the keys and the first few over queries and values
  // (head n of those: query n, then value n - nq)
  const int rest = a.nq + nkv;
  HalfPair k_raw = {}, raw[kAppendAhead] = {};
  if (lh < nkv) k_raw = load(row + (a.nq + lh) * HD);
  auto request = [&](int n0) {
#pragma unroll
    for (int i = 0; i < kAppendAhead; ++i) {
      const int n = n0 + i * PH + lh;
      if (n < rest) raw[i] = load(row + (n < a.nq ? n : n + nkv) * HD);
    }
  };
  request(0);
  if (slot >= a.kv.n_pages * a.kv.page_size) {
    if (threadIdx.x == 0 && p >= 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    slot = -1;
  }
  if (slot < 0 || p < 0) {
    uint4* q = reinterpret_cast<uint4*>(a.q_out + (size_t)t * a.nq * HD);
    for (int i = threadIdx.x; i < a.nq * L; i += kAppendThreads)
      q[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x < HD / 2) {
    double turns = (double)p * freq * 0.15915494309189533577;  // / (2 pi)
    turns -= rint(turns);
    float2 r;
    sincospif((float)(2.0 * turns), &r.y, &r.x);
    s_rot[threadIdx.x] = r;
    if constexpr (E4M3) sincospi(2.0 * turns, &s_rot_k[threadIdx.x].y, &s_rot_k[threadIdx.x].x);
  }
  __syncthreads();
  float2 rot[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) rot[j] = s_rot[4 * l + j];
  // a lane's share of a head in type R: RMSNorm (by(mean square) is the
  // factor), then the rotation
  auto rotated = [&](auto zero, const HalfPair& in, const HalfPair& weight, const auto* ro,
                     float (&u)[4], float (&v)[4], auto by) {
    using R = decltype(zero);
    R x[4], y[4], wx[4], wy[4], ss = zero;
    in.get(x, y);
    weight.get(wx, wy);
#pragma unroll
    for (int j = 0; j < 4; ++j) ss += x[j] * x[j] + y[j] * y[j];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const R f = by(ss / (R)HD + (R)a.eps);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const R n = x[j] * f * wx[j], m = y[j] * f * wy[j];
      u[j] = (float)(n * ro[j].x - m * ro[j].y);
      v[j] = (float)(n * ro[j].y + m * ro[j].x);
    }
  };
  auto half = [](const float (&x)[4]) {
    return make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
  };
  const int page = slot >> a.kv.page_shift, off = slot & (a.kv.page_size - 1);
  auto put = [&](const float (&u)[4], const float (&v)[4], int kh, int is_v) {
    const size_t at =
        (((((size_t)page * 2 + is_v) * nkv + kh) << a.kv.page_shift) + off) * HD + 4 * l;
    if constexpr (E4M3) {
      *reinterpret_cast<uint32_t*>(a.kv.base + at) = f32x4_to_e4m3(u);
      *reinterpret_cast<uint32_t*>(a.kv.base + at + HD / 2) = f32x4_to_e4m3(v);
    } else {
      *reinterpret_cast<uint2*>(a.kv.base + 2 * at) = half(u);
      *reinterpret_cast<uint2*>(a.kv.base + 2 * at + HD) = half(v);
    }
  };
  float u[4], v[4];
  for (int h0 = 0; h0 < nkv; h0 += PH) {
    const int h = h0 + lh;
    // (warps without a key have nothing to sum)
    if (!__any_sync(0xffffffffu, h < nkv)) continue;
    if (h0 > 0 && h < nkv) k_raw = load(row + (a.nq + h) * HD);
    if constexpr (E4M3)
      rotated(0.0, k_raw, wk, s_rot_k + 4 * l, u, v, [&](double ms) {
        return rsqrt(ms) / (double)(h < nkv ? a.kv.k_scale[h] : 1.f);
      });
    else
      rotated(0.f, k_raw, wk, rot, u, v, [](float ms) { return rsqrtf(ms); });
    if (h < nkv) put(u, v, h, 0);
  }
  for (int n0 = 0; n0 < rest; n0 += kAppendAhead * PH) {
    if (n0 > 0) request(n0);
#pragma unroll
    for (int i = 0; i < kAppendAhead; ++i) {
      const int n = n0 + i * PH + lh;
      if (__any_sync(0xffffffffu, n < a.nq)) {
        rotated(0.f, raw[i], wq, rot, u, v, [](float ms) { return rsqrtf(ms); });
        if (n < a.nq) {
          uint2* q = reinterpret_cast<uint2*>(a.q_out + ((size_t)t * a.nq + n) * HD);
          q[l] = half(u);
          q[l + L] = half(v);
        }
      }
      if (n >= a.nq && n < rest) {
        raw[i].get(u, v);
        if constexpr (E4M3) {
          const float sc = a.kv.v_scale[n - a.nq];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            u[j] /= sc;
            v[j] /= sc;
          }
        }
        put(u, v, n - a.nq, 1);
      }
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
//   S^T [16 keys x 8 cols] = K [16 x hd] q^T,   O^T [hd x 8] += V^T P^T
// with mma.m16n8k16: M is keys / dims, so no row is padding (tcgen05's
// smallest M of 64 or 128 heads would be).  The columns are the q heads of
// one row and, where they leave room, of the rows after it that belong to the
// same request (a prompt's rows share their keys: see lead_keys; calls whose
// requests have many rows go to slx_paged_tile.cu).
//
// The contraction index of an MMA may be permuted on both sides alike; the
// fragments are chosen so that each is 16 contiguous bytes of a key.
//   bf16: keys and values go from global memory to fragments without shared
//   memory, the next unit's into the registers that this one's have just left
//   (256 requests of 6k tokens, 24/4 heads, in a graph: 473 to 482 us by the
//   machine, 6.8 to 6.95 TB/s, where a copy's reads and writes reach 6.5; through
//   the ring below 499).
//   e4m3: half the bytes and twice the work per byte.  A unit's keys and its
//   values are one contiguous block each: every warp has a ring of stages in
//   shared memory that its first lane fills by bulk copies, some units ahead
//   and across the ends of rows (128 requests of 1k to 16k tokens, 16/2 heads, in
//   a graph: 108 to 121 us by the machine; with register loads 134 where this
//   took 111).
// V pairs two keys per register (byte permutes); S^T's accumulators become
// P^T's operand by movmatrix.
//
// P is rounded to two 16-bit parts, hi + lo.  For bf16 pages they are bf16: 16
// bits of any weight, so the only rounding of note is the output's.  For e4m3
// pages they are fp16, whose range P is shifted to the top of: the greatest
// weight is 2^15, one of 2^-29 of it still has 11 bits, and the least step is
// 2^-39 of it, so a result is off by 2^-40 sum |v| at most.  E4m3 keys and values
// become fp16 exactly; q becomes fp16 times a power of two per head that puts
// its largest element at 2^12 .. 2^13 (exact down to 2^-26 of it).
//
// Work is cut into units of one kv head (16 bf16 or 32 e4m3 keys); every CTA
// gets an equal share of the list (row group, kv head, unit), whatever the
// rows' lengths.  A segment, the units of one (group, kv head), weighs
// kPaSwitch units more than it has, about what the change to it costs (64
// requests of 0 to 4k tokens, in a graph: 51 us, 59 without).  A segment that one CTA
// covers is written directly, the others leave (max, sum, O) parts that
// k_paged_join adds in order.

constexpr int kPaWarps = 4;
constexpr int kPaThreads = 32 * kPaWarps;
constexpr int kPaStages = 2;  // of a warp's ring
constexpr int kPaSwitch = 8;  // units
// 16-key halves of a unit: as many bytes in flight either way
constexpr int pa_halves(bool e4m3) { return e4m3 ? 2 : 1; }
// P and its sum are 2^kPaUp times the softmax's (the quotient is not): with fp16
// parts as high as its range of 65504 allows
template <bool E4M3>
constexpr float kPaUp = E4M3 ? 15.f : 0.f;

struct PaWork {       // workspace of one call
  int4* desc;         // [n] split (group, kv head): first, last CTA, row, head
  float* o;           // [2 CTAs][cols][hd] parts: 2 w + 1 a segment's first
  float2* ml;         // [2 CTAs][cols] max (log2), sum; sum -1: no such row
};

SLX_DEV void ld_stream(const uint8_t* p, uint32_t* v) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "l"(p));
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

// Rows are taken in aligned blocks of `rpb` (a power of two up to 16: what fits
// the MMA's columns); within one, consecutive rows of the same request form a group.
// For a warp over rows t0 .. t0 + 31 (t0 a multiple of 32; n and r its rows'
// keys and requests): the keys of the group that row t0 + lane leads, 0 if it
// leads none.
SLX_DEV int lead_keys(int n, int r, int rpb) {
  if (rpb == 1) return n;
  const int lane = threadIdx.x & 31;
  const int before = __shfl_up_sync(0xffffffffu, r, 1);
  const bool first = lane % rpb == 0 || before != r;
  const unsigned starts = __ballot_sync(0xffffffffu, first);
  const unsigned behind = lane == 31 ? 0u : starts >> (lane + 1);
  const int end = behind ? lane + __ffs(behind) : 32;  // of this lane's group
  int most = n;
  for (int d = 1; d < rpb; d <<= 1) {
    const int v = __shfl_down_sync(0xffffffffu, most, d);
    if (lane + d < end) most = max(most, v);
  }
  return first ? most : 0;
}

// Sum of 0 <= n < 2^28 over a warp.
SLX_DEV long long warp_sum(int n) {
  return (long long)__reduce_add_sync(0xffffffffu, (unsigned)n & 0xffffu) +
         ((long long)__reduce_add_sync(0xffffffffu, (unsigned)n >> 16) << 16);
}

// A run of units of one (row group, kv head) that falls to this CTA.
struct PaSeg {
  int row, kh, u0, u1, units, keys, req;
};

// REST: behind k_paged_tile, for the rows that it has left.
template <int HD, bool E4M3, int NT, bool REST>
__global__ void __launch_bounds__(kPaThreads, HD == 64 ? 5 - NT : 4 - NT)
    k_paged_attn(const PagedAttnArgs a, const PaWork ws, int rpb, const TileWork tile) {
  constexpr int ES = E4M3 ? 1 : 2;       // bytes per element
  constexpr int RB = HD * ES;            // a key's row
  constexpr int KQ = RB / 64;            // 16-byte pieces of a key per lane
  constexpr int KS = HD / 16;            // MMA steps of q . k
  constexpr int MT = HD / 16;            // 16-dim tiles of O^T
  constexpr int VB = RB >= 128 ? 16 : 8; // bytes of a piece of V
  constexpr int VP = RB / (8 * VB);      // its pieces per key
  constexpr int VW = RB / 32;            // words per lane and key
  constexpr bool RING = E4M3;
  constexpr int H = pa_halves(E4M3), kPaUnit = 16 * H;
  constexpr int SB = 2 * kPaUnit * RB;   // a unit's keys, then its values
  constexpr int S = RING ? kPaStages : 1;
  extern __shared__ __align__(128) uint8_t pa_smem[];
  // merging the warps' states: two of them at a time, as they lie in registers
  float4* s_acc = reinterpret_cast<float4*>(pa_smem + (RING ? kPaWarps * S * SB : 0));
  __shared__ __align__(8) uint64_t s_bar[kPaWarps][S];
  __shared__ int s_bad[kPaWarps][S];     // halves of the stage without a page
  __shared__ float s_ml[2][2][8 * NT];
  __shared__ long long s_pre[kPaThreads + 1];
  __shared__ long long w_sum[kPaWarps];
  __shared__ int s_run;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int w = blockIdx.x, nw = gridDim.x;
  const int nkv = a.kv.n_kv, G = a.nq / nkv, ps = a.kv.page_size;
  const int cols = rpb * G;
  const int sh = a.kv.page_shift;
  const bool by_row = (long long)a.T * nkv <= nw;  // how desc is indexed
  pdl_launch_dependents();
  pdl_wait_primary();
  if constexpr (REST) {
    if (tile.n_left) {
      int any = 0;
      for (int i = tid; i < tile.n_left; i += kPaThreads) any |= tile.left[i];
      if (!__syncthreads_or(any)) {
        if (tid == 0) ws.desc[w] = make_int4(-1, 0, 0, 0);
        return;
      }
    }
  }
  // the keys of the group that row t0 + lane leads and that falls to this kernel
  auto lead = [&](const RowKeys& r, int t0) {
    const int n = lead_keys(r.keys, r.req, rpb);
    if constexpr (REST) return in_run(a, t0, tile.least) ? 0 : n;
    return n;
  };
  auto units_of = [](int keys) { return (int)(((unsigned)keys + kPaUnit - 1) / kPaUnit); };
  auto weight_of = [&](int keys) { return keys ? units_of(keys) + kPaSwitch : 0; };
  // weights before each of 128 runs of `run` tiles of 32 rows
  const int tiles = (a.T + 31) / 32, run = (tiles + kPaThreads - 1) / kPaThreads;
  RowKeys rk;                             // of row rb + lane
  int len_l = 0;                          // keys of the group it leads
  long long total;
  if (tiles == 1) {
    rk = row_keys(a, lane);
    len_l = lead(rk, 0);
    total = warp_sum(weight_of(len_l)) * nkv;
  } else {
    s_pre[tid + 1] = 0;
    __syncthreads();
    constexpr int B = 4;  // tiles whose rows are read together
    for (int i0 = warp * B; i0 < tiles; i0 += B * kPaWarps) {
      RowKeys r[B];
#pragma unroll
      for (int j = 0; j < B; ++j) r[j] = row_keys(a, (i0 + j) * 32 + lane);
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const long long v = warp_sum(weight_of(lead(r[j], (i0 + j) * 32)));
        if (lane == 0 && i0 + j < tiles)
          atomicAdd(reinterpret_cast<unsigned long long*>(&s_pre[(i0 + j) / run + 1]),
                    (unsigned long long)v);
      }
    }
    __syncthreads();
    long long v = s_pre[tid + 1];
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
    __syncthreads();
    total = s_pre[kPaThreads] * nkv;
  }
  // weight per CTA: a multiple of the warps (a step is one unit per warp)
  long long per = total < 0x7fffffff - nw ? ((unsigned)total + nw - 1) / (unsigned)nw
                                          : (total + nw - 1) / nw;
  per = (per + kPaWarps - 1) / kPaWarps * kPaWarps;
  if (per < kPaWarps) per = kPaWarps;
  long long x = w * per;
  const long long x_end = min(x + per, total);
  int4 my_desc = make_int4(-1, 0, 0, 0);
  if (x < x_end) {
    PaSeg sg;
    int rb = 0;
    {
      // the segment x is in: its run of tiles, then tile by tile
      long long before = 0;
      if (tiles > 1) {
        if (s_pre[tid] * nkv <= x && x < s_pre[tid + 1] * nkv) s_run = tid;
        __syncthreads();
        rb = s_run * run * 32;
        before = s_pre[s_run] * nkv;
      }
      for (;; rb += 32) {
        if (tiles > 1) {
          rk = row_keys(a, rb + lane);
          len_l = lead(rk, rb);
        }
        const int n = weight_of(len_l);
        const long long all = warp_sum(n);
        if (x >= before + all * nkv) {
          before += all * nkv;
          continue;
        }
        // the row whose weights (times nkv) reach beyond x
        auto find = [&](auto v, auto in) {
          const auto own = v;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const auto u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
          }
          const int i = __ffs(__ballot_sync(0xffffffffu, v > in)) - 1;
          sg.row = rb + i;
          before += (long long)__shfl_sync(0xffffffffu, v - own, i) * nkv;
          return i;
        };
        const long long in = x - before < 0x7fffffff ? (unsigned)(x - before) / (unsigned)nkv
                                                     : (x - before) / nkv;
        const int i = all < 0x7fffffff ? find(n, (int)in) : find((long long)n, in);
        sg.keys = __shfl_sync(0xffffffffu, len_l, i);
        sg.req = __shfl_sync(0xffffffffu, rk.req, i);
        break;
      }
      sg.units = units_of(sg.keys);
      const int weight = sg.units + kPaSwitch;
      const long long in = x - before;
      sg.kh = in < 0x7fffffff ? (int)((unsigned)in / (unsigned)weight) : (int)(in / weight);
      before += (long long)sg.kh * weight + kPaSwitch;  // of the segment's first unit
      sg.u0 = (int)max(x - before, 0LL);
      sg.u1 = (int)max(min((long long)sg.units, x_end - before), 0LL);
      x = before;
    }
    const size_t page_bytes = (size_t)2 * nkv * ps * RB, v_off = (size_t)nkv * ps * RB;
    // a place in the CTA's segments: the rows of tile rb and x as above
    struct Place {
      PaSeg sg;
      int rb, len, req;  // len, req: of row rb + lane
      long long x;       // the place of the segment's first unit
    };
    // to the next segment; false behind the last
    auto advance = [&](Place& p) {
      p.x += p.sg.units + kPaSwitch;
      if (p.x >= x_end) return false;
      p.sg.u0 = 0;
      if (++p.sg.kh == nkv) {
        p.sg.kh = 0;
        unsigned hit = __ballot_sync(0xffffffffu, p.len > 0 && p.rb + lane > p.sg.row);
        while (!hit) {  // there is one: x < total
          p.rb += 32;
          const RowKeys r = row_keys(a, p.rb + lane);
          p.len = lead(r, p.rb);
          p.req = r.req;
          hit = __ballot_sync(0xffffffffu, p.len > 0);
        }
        const int i = __ffs(hit) - 1;
        p.sg.row = p.rb + i;
        p.sg.keys = __shfl_sync(0xffffffffu, p.len, i);
        p.sg.req = __shfl_sync(0xffffffffu, p.req, i);
        p.sg.units = units_of(p.sg.keys);
      }
      p.sg.u1 = (int)min((long long)p.sg.units, x_end - p.x);
      return true;
    };
    Place at = {sg, rb, len_l, rk.req, x};   // what is computed
    uint32_t vr[4][VW];  // words of values 2c, 2c + 1, 2c + 8, 2c + 9
    // ---- register loads (bf16; units of 16 keys)
    uint32_t kr[RING ? 1 : 2][KQ][4];        // pieces of keys g, g + 8
    // page of unit u of the current segment
    auto page_of = [&](int u) {
      return u < at.sg.u1 ? a.table[(size_t)at.sg.req * a.max_pages + ((u * kPaUnit) >> sh)] : -1;
    };
    auto keys_at = [&](int u, int page) {
      return a.kv.base + (size_t)(unsigned)page * page_bytes +
             ((size_t)at.sg.kh * ps + ((u * kPaUnit) & (ps - 1))) * RB;
    };
    // the unit's last key that the group holds, -1 for a page out of range
    auto last_of = [&](int u, int page) {
      if ((unsigned)page < (unsigned)a.kv.n_pages)
        return min(kPaUnit, at.sg.keys - u * kPaUnit) - 1;
      if (lane == 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      return -1;
    };
    auto load_k = [&](int u, int page) {
      if constexpr (!RING) {
        const int last = last_of(u, page);
        const uint8_t* p = keys_at(u, last < 0 ? 0 : page) + g * RB + c * 16;
        if (last == kPaUnit - 1) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int q = 0; q < KQ; ++q) ld_stream(p + r * 8 * RB + q * 64, kr[r][q]);
        } else {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int q = 0; q < KQ; ++q) {
              kr[r][q][0] = kr[r][q][1] = kr[r][q][2] = kr[r][q][3] = 0;
              if (g + 8 * r <= last) ld_stream(p + r * 8 * RB + q * 64, kr[r][q]);
            }
        }
      }
    };
    auto load_v = [&](int u, int page) {
      if constexpr (!RING) {
        const int last = last_of(u, page);
        const uint8_t* p = keys_at(u, last < 0 ? 0 : page) + v_off + 2 * c * RB + g * VB;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = (r & 1) + 8 * (r >> 1);
          if (last < kPaUnit - 1) {
#pragma unroll
            for (int q = 0; q < VW; ++q) vr[r][q] = 0;
            if (2 * c + key > last) continue;
          }
#pragma unroll
          for (int q = 0; q < VP; ++q) ld_stream(p + key * RB + q * 128, vr[r] + q * 4);
        }
      }
    };
    int page = RING ? -1 : page_of(sg.u0 + warp);
    bool loaded = false;                     // the segment's first unit is on its way
    // ---- ring of bulk copies (e4m3)
    Place ahead = at;                        // what is requested
    uint8_t* ring = pa_smem + warp * (S * SB);
    if (RING && lane == 0) {
#pragma unroll
      for (int i = 0; i < S; ++i) mbar_init(&s_bar[warp][i], 1);
      fence_mbar_init();
    }
    __syncwarp();
    int next_u = sg.u0 + warp, next_page[H];
    bool live = true;
    // this warp's next unit to request, and its page
    auto seek = [&] {
      while (next_u >= ahead.sg.u1) {
        if (!advance(ahead)) {
          live = false;
          return;
        }
        next_u = warp;
      }
      const int32_t* tab = a.table + (size_t)ahead.sg.req * a.max_pages;
      const int k0 = next_u * kPaUnit;
      next_page[0] = tab[k0 >> sh];
      // (a page of 16 keys is half a unit of 32)
      if constexpr (H == 2)
        next_page[1] = ps > 16 ? next_page[0] : k0 + 16 < ahead.sg.keys ? tab[(k0 + 16) >> sh] : 0;
    };
    auto request = [&](int st) {
      if (!live) return;
      if (lane == 0) {
        const PaSeg& s = ahead.sg;
        const int k0 = next_u * kPaUnit, held = min(kPaUnit, s.keys - k0);
        uint64_t* bar = &s_bar[warp][st];
        uint8_t* dst = ring + st * SB;
        auto block = [&](int page, int k) {
          return a.kv.base + (size_t)page * page_bytes +
                 ((size_t)s.kh * ps + (k & (ps - 1))) * RB;
        };
        const bool one = H == 1 || ps > 16;     // the unit lies on one page
        int bad = 0;
#pragma unroll
        for (int h = 0; h < H; ++h)
          if ((unsigned)next_page[h] >= (unsigned)a.kv.n_pages) bad |= 1 << h;
        s_bad[warp][st] = bad;
        if (bad) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
        if (one && !bad) {
          mbar_arrive_expect_tx(bar, 2 * held * RB);
          const uint8_t* src = block(next_page[0], k0);
          bulk_g2s_plain(dst, src, held * RB, bar);
          bulk_g2s_plain(dst + kPaUnit * RB, src + v_off, held * RB, bar);
        } else {
          const int n0 = bad & 1 ? 0 : min(held, 16), n1 = one || (bad & 2) ? 0 : max(held - 16, 0);
          mbar_arrive_expect_tx(bar, 2 * (n0 + n1) * RB);
          if (n0) {
            const uint8_t* src = block(next_page[0], k0);
            bulk_g2s_plain(dst, src, n0 * RB, bar);
            bulk_g2s_plain(dst + kPaUnit * RB, src + v_off, n0 * RB, bar);
          }
          if (n1) {
            const uint8_t* src = block(next_page[H - 1], k0 + 16);
            bulk_g2s_plain(dst + 16 * RB, src, n1 * RB, bar);
            bulk_g2s_plain(dst + (kPaUnit + 16) * RB, src + v_off, n1 * RB, bar);
          }
        }
      }
      next_u += kPaWarps;
      seek();
    };
    int used = 0;                            // units this warp has taken from it
    if constexpr (RING) {
      seek();
#pragma unroll
      for (int i = 0; i < S; ++i) request(i);
    }
    // (a CTA whose share ends before a first unit computes nothing)
    while (at.sg.u1 > at.sg.u0) {
      sg = at.sg;
      int u = sg.u0 + warp;
      // columns n of the MMAs: row n / G of the group, q head n % G
      uint32_t qf[NT][KS][2];
      float fac[NT][2];  // of columns 2c, 2c + 1: scores in log2 units
      int lim[NT][2];    // their keys (0: no such row)
      const float fs = a.scale * 1.4426950408889634f * (E4M3 ? a.kv.k_scale[sg.kh] : 1.f);
      uint4 qv[NT][HD / 32];
      int rows = rpb;    // of the group
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int n = nt * 8 + g;
        int row = sg.row, keys = n < cols ? sg.keys : 0;
        if (rpb > 1) {
          // the group ends before its first row of another request or block
          row += n / G;
          const RowKeys r = row_keys(a, row);
          const bool on = row < a.T && row / rpb == sg.row / rpb && r.req == sg.req;
          rows = min(rows, (int)__reduce_min_sync(0xffffffffu, on ? rpb : n / G));
          keys = n < cols && n / G < rows ? r.keys : 0;
        }
        lim[nt][0] = __shfl_sync(0xffffffffu, keys, 8 * c);
        lim[nt][1] = __shfl_sync(0xffffffffu, keys, 8 * c + 4);
        const uint8_t* qp = reinterpret_cast<const uint8_t*>(
            a.q + (size_t)(keys ? row : sg.row) * a.q_stride +
            (size_t)(sg.kh * G + n % G) * HD);
        // bf16 pages: 8 dims of each 32; e4m3: 16 of each 64 (as the keys')
#pragma unroll
        for (int q = 0; q < HD / 32; ++q)
          qv[nt][q] = keys > 0 ? *reinterpret_cast<const uint4*>(
                                     qp + (E4M3 ? (q >> 1) * 128 + c * 32 + (q & 1) * 16
                                                : q * 64 + c * 16))
                               : make_uint4(0, 0, 0, 0);
      }
      if constexpr (!RING) {
        if (u < sg.u1 && !loaded) {
          load_k(u, page);
          load_v(u, page);
        }
        page = page_of(u + kPaWarps);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (!E4M3) {
#pragma unroll
          for (int q = 0; q < HD / 32; ++q) {
            qf[nt][2 * q][0] = qv[nt][q].x;
            qf[nt][2 * q][1] = qv[nt][q].y;
            qf[nt][2 * q + 1][0] = qv[nt][q].z;
            qf[nt][2 * q + 1][1] = qv[nt][q].w;
          }
          fac[nt][0] = fac[nt][1] = fs;
        } else {
          float mx = 0.f;
#pragma unroll
          for (int q = 0; q < HD / 32; ++q) {
            const uint32_t v[4] = {qv[nt][q].x, qv[nt][q].y, qv[nt][q].z, qv[nt][q].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(v[i])), fabsf(bf16_hi(v[i]))));
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // 2^k: the largest element lands in [2^12, 2^13)
          const int e = (int)(__float_as_uint(mx) >> 23) - 127;
          const int k = mx == 0.f || e == 128 ? 0 : min(12 - e, 100);
          const float up = __uint_as_float((uint32_t)(127 + k) << 23);
          const float down = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
          for (int q = 0; q < HD / 32; ++q) {
            const uint32_t v[4] = {qv[nt][q].x, qv[nt][q].y, qv[nt][q].z, qv[nt][q].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              qf[nt][2 * q + (i >> 1)][i & 1] = pack_f16x2(bf16_lo(v[i]) * up, bf16_hi(v[i]) * up);
          }
          // lane 8c holds column 2c's factor, lane 8c + 4 column 2c + 1's
          fac[nt][0] = fs * __shfl_sync(0xffffffffu, down, 8 * c);
          fac[nt][1] = fs * __shfl_sync(0xffffffffu, down, 8 * c + 4);
        }
      }
      // keys that every row of the group attends
      int common = sg.keys;
      if (rpb > 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (lim[nt][i]) common = min(common, lim[nt][i]);
        common = __reduce_min_sync(0xffffffffu, common);
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
      for (; u < sg.u1; u += kPaWarps) {
        const int k0 = u * kPaUnit, st = used % S;
        int bad = 0;                         // halves of the unit without a page
        if constexpr (RING) {
          mbar_wait(&s_bar[warp][st], used / S & 1, a.status);
          bad = s_bad[warp][st];
          ++used;
        }
        const uint8_t* sk = ring + st * SB + g * RB + c * 16;
        const uint8_t* sv = ring + st * SB + kPaUnit * RB + 2 * c * RB + g * VB;
        float s[NT][H][4];
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float s2[NT][4];  // even and odd steps: two shorter chains
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][h][i] = s2[nt][i] = 0.f;
#pragma unroll
          for (int q = 0; q < KQ; ++q) {
            uint32_t lo[4], hi[4];  // pieces of keys g, g + 8
            if constexpr (RING) {
              const uint4 x0 = *reinterpret_cast<const uint4*>(sk + 16 * h * RB + q * 64);
              const uint4 x1 = *reinterpret_cast<const uint4*>(sk + (16 * h + 8) * RB + q * 64);
              lo[0] = x0.x; lo[1] = x0.y; lo[2] = x0.z; lo[3] = x0.w;
              hi[0] = x1.x; hi[1] = x1.y; hi[2] = x1.z; hi[3] = x1.w;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                lo[i] = kr[0][q][i];
                hi[i] = kr[RING ? 0 : 1][q][i];
              }
            }
            if constexpr (!E4M3) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<true>(s[nt][h], lo[0], hi[0], lo[1], hi[1], qf[nt][2 * q][0],
                               qf[nt][2 * q][1]);
                mma16816<true>(s2[nt], lo[2], hi[2], lo[3], hi[3], qf[nt][2 * q + 1][0],
                               qf[nt][2 * q + 1][1]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t a0, a1, a2, a3;
                e4m3x4(lo[i], a0, a2);
                e4m3x4(hi[i], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816<false>(i & 1 ? s2[nt] : s[nt][h], a0, a1, a2, a3,
                                  qf[nt][4 * q + i][0], qf[nt][4 * q + i][1]);
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s[nt][h][i] = (s[nt][h][i] + s2[nt][i]) * fac[nt][i & 1];
              // a page out of range holds zeros
              if (bad >> h & 1) s[nt][h][i] = 0.f;
            }
        }
        const bool more_u = u + kPaWarps < sg.u1;
        const int pg = page;
        if (!RING && more_u) {
          load_k(u + kPaWarps, pg);
          page = page_of(u + 2 * kPaWarps);
        }
        uint32_t ph[NT][H][2], pl[NT][H][2];  // P^T operands: hi and lo parts
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (k0 + kPaUnit > common) {
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (k0 + 16 * h + 8 * (i >> 1) + g >= lim[nt][i & 1]) s[nt][h][i] = -INFINITY;
          }
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = fmaxf(s[nt][0][i], s[nt][0][i + 2]);
            if constexpr (H == 2) mx = fmaxf(mx, fmaxf(s[nt][H - 1][i], s[nt][H - 1][i + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[nt][i]);
            const float ms = mx == -INFINITY ? 0.f : mx, mt = ms - kPaUp<E4M3>;
            f[i] = exp2_fast(m[nt][i] - ms);
            m[nt][i] = mx;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < H; ++h) {
              s[nt][h][i] = exp2_fast(s[nt][h][i] - mt);
              s[nt][h][i + 2] = exp2_fast(s[nt][h][i + 2] - mt);
              sum += s[nt][h][i] + s[nt][h][i + 2];
            }
            l[nt][i] = l[nt][i] * f[i] + sum;
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
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float p0 = s[nt][h][2 * r], p1 = s[nt][h][2 * r + 1];
              uint32_t hi, lo;
              if constexpr (!E4M3) {
                hi = pack_bf16(p0, p1);
                lo = pack_bf16(p0 - bf16_lo(hi), p1 - bf16_hi(hi));
              } else {
                hi = pack_f16x2(p0, p1);
                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                lo = pack_f16x2(p0 - b.x, p1 - b.y);
              }
              ph[nt][h][r] = transpose8x8(hi);
              pl[nt][h][r] = transpose8x8(lo);
            }
        }
        // V^T fragments of tile i
        auto frag = [&](int i, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3,
                        uint32_t (&f)[4]) {
          if constexpr (!E4M3) {
            // word i of the lane's dims: dims 2i (low halves) and 2i + 1
            f[0] = __byte_perm(v0, v1, 0x5410);
            f[1] = __byte_perm(v0, v1, 0x7632);
            f[2] = __byte_perm(v2, v3, 0x5410);
            f[3] = __byte_perm(v2, v3, 0x7632);
          } else {
            // bytes 2 (i % 2), + 1 of word i / 2: dims 2i and 2i + 1
            const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
            e4m3x4(__byte_perm(v0, v1, sel), f[0], f[1]);
            e4m3x4(__byte_perm(v2, v3, sel), f[2], f[3]);
          }
        };
        constexpr int D = E4M3 ? 2 : 1;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int kh0 = k0 + 16 * h;
          if constexpr (RING) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int q = 0; q < VP; ++q) {
                const uint8_t* p = sv + (16 * h + (r & 1) + 8 * (r >> 1)) * RB + q * 128;
                if constexpr (VB == 16) {
                  const uint4 v = *reinterpret_cast<const uint4*>(p);
                  vr[r][4 * q] = v.x;
                  vr[r][4 * q + 1] = v.y;
                  vr[r][4 * q + 2] = v.z;
                  vr[r][4 * q + 3] = v.w;
                } else {
                  const uint2 v = *reinterpret_cast<const uint2*>(p);
                  vr[r][0] = v.x;
                  vr[r][1] = v.y;
                }
              }
            if (h == H - 1) {
              __syncwarp();  // the stage is read: refill it
              request(st);
            }
            // behind the group's keys the stage holds an earlier unit's values
            if ((bad >> h & 1) || kh0 + 16 > sg.keys) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if ((bad >> h & 1) || kh0 + 2 * c + (r & 1) + 8 * (r >> 1) >= sg.keys) {
#pragma unroll
                  for (int q = 0; q < VW; ++q) vr[r][q] = 0;
                }
            }
          }
          // a weight of 0 does not hide an infinite or NaN value from a row
          // that does not attend it: such keys go row by row
          bool apart = false;
          if (rpb > 1 && kh0 + 16 > common) {
            bool odd = false;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int q = 0; q < VW; ++q) {
                const uint32_t v = vr[r][q];
                if constexpr (!E4M3)
                  odd |= (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
                else
                  odd |= ((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
              }
            apart = __any_sync(0xffffffffu, odd);
          }
          if (!apart) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              uint32_t f[4];
              frag(i, vr[0][i / D], vr[1][i / D], vr[2][i / D], vr[3][i / D], f);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<!E4M3>(acc[nt][i], f[0], f[1], f[2], f[3], ph[nt][h][0], ph[nt][h][1]);
                mma16816<!E4M3>(acc[nt][i], f[0], f[1], f[2], f[3], pl[nt][h][0], pl[nt][h][1]);
              }
            }
          } else {
#pragma unroll 1
            for (int j = 0; j < rpb; ++j) {
              const int row = sg.row + j;
              const RowKeys rj = row_keys(a, row);
              if (row >= a.T || row / rpb != sg.row / rpb || rj.req != sg.req) break;
              const int at = kh0 + 2 * c, keys = rj.keys;
              const bool on[4] = {at < keys, at + 1 < keys, at + 8 < keys, at + 9 < keys};
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                uint32_t f[4];
                frag(i, on[0] ? vr[0][i / D] : 0, on[1] ? vr[1][i / D] : 0,
                     on[2] ? vr[2][i / D] : 0, on[3] ? vr[3][i / D] : 0, f);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  float t[4] = {0.f, 0.f, 0.f, 0.f};
                  mma16816<!E4M3>(t, f[0], f[1], f[2], f[3], ph[nt][h][0], ph[nt][h][1]);
                  mma16816<!E4M3>(t, f[0], f[1], f[2], f[3], pl[nt][h][0], pl[nt][h][1]);
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    if ((nt * 8 + 2 * c + (k & 1)) / G == j) acc[nt][i][k] += t[k];
                }
              }
            }
          }
        }
        if (!RING && more_u) load_v(u + kPaWarps, pg);
      }
      const long long x0 = at.x;
      const bool more = advance(at);
      if (!RING && more) page = page_of(warp);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], 4);
          l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], 8);
          l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], 16);
        }
      // warps 2, 3 into 0, 1, then 1 into 0
#pragma unroll
      for (int half = kPaWarps / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp >= half && warp < 2 * half) {
          float4* d = s_acc + (warp - half) * (NT * MT * 32) + lane;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
              d[(nt * MT + i) * 32] = make_float4(acc[nt][i][0], acc[nt][i][1],
                                                  acc[nt][i][2], acc[nt][i][3]);
            if (g == 0) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                s_ml[warp - half][0][nt * 8 + 2 * c + i] = m[nt][i];
                s_ml[warp - half][1][nt * 8 + 2 * c + i] = l[nt][i];
              }
            }
          }
        }
        __syncthreads();
        if (!RING && half == kPaWarps / 2) {
          // the next segment's first unit, while the states are merged
          loaded = more && warp < at.sg.u1;
          if (loaded) {
            load_k(warp, page);
            load_v(warp, page);
          }
        }
        if (warp < half) {
          const float4* d = s_acc + warp * (NT * MT * 32) + lane;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float f0[2], f1[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float om = s_ml[warp][0][nt * 8 + 2 * c + i];
              const float mx = fmaxf(m[nt][i], om);
              const float ms = mx == -INFINITY ? 0.f : mx;
              f0[i] = exp2_fast(m[nt][i] - ms);
              f1[i] = exp2_fast(om - ms);
              l[nt][i] = l[nt][i] * f0[i] + s_ml[warp][1][nt * 8 + 2 * c + i] * f1[i];
              m[nt][i] = mx;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const float4 v = d[(nt * MT + i) * 32];
              acc[nt][i][0] = acc[nt][i][0] * f0[0] + v.x * f1[0];
              acc[nt][i][1] = acc[nt][i][1] * f0[1] + v.y * f1[1];
              acc[nt][i][2] = acc[nt][i][2] * f0[0] + v.z * f1[0];
              acc[nt][i][3] = acc[nt][i][3] * f0[1] + v.w * f1[1];
            }
          }
        }
      }
      const bool whole = sg.u0 == 0 && sg.u1 == sg.units;
      if (warp == 0) {
        const float sv = E4M3 ? a.kv.v_scale[sg.kh] : 1.f;
        const size_t part = 2 * (size_t)w + (sg.u0 == 0 ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int n = nt * 8 + 2 * c + i;
            if (n >= cols) continue;
            const float scale = whole ? sv / l[nt][i] : sv;
            float* po = ws.o + (part * cols + n) * HD;
            uint16_t* out = a.out + ((size_t)(sg.row + n / G) * a.nq + sg.kh * G + n % G) * HD;
            if (!whole && g == 0)
              ws.ml[part * cols + n] = make_float2(m[nt][i], lim[nt][i] ? l[nt][i] : -1.f);
            if (lim[nt][i] == 0) continue;  // no such row
#pragma unroll
            for (int j = 0; j < MT; j += 2) {
              // tiles j, j + 1: four consecutive dims
              const int d = E4M3 ? g * (HD / 8) + 2 * j : (j / 4) * 64 + g * 8 + (j % 4) * 2;
              const float4 o = make_float4(acc[nt][j][i] * scale, acc[nt][j][i + 2] * scale,
                                           acc[nt][j + 1][i] * scale,
                                           acc[nt][j + 1][i + 2] * scale);
              if (whole)
                *reinterpret_cast<uint2*>(out + d) =
                    make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
              else
                *reinterpret_cast<float4*>(po + d) = o;
            }
          }
      }
      if (sg.u0 == 0) {
        const int4 d = whole ? make_int4(-1, 0, 0, 0)
                             : make_int4(w, (int)((x0 + sg.units - 1) / per), sg.row, sg.kh);
        if (by_row) {
          if (tid == 0) ws.desc[sg.row * nkv + sg.kh] = d;
        } else if (!whole) {
          my_desc = d;
        }
      }
      if (!more) break;
    }
  }
  if (!by_row && tid == 0) ws.desc[w] = my_desc;
  // idle rows: zeros (and the status of those out of range)
  if (warp != 0) return;
  for (int i = w; i < tiles; i += nw) {
    const int t = i * 32 + lane;
    const RowKeys r = row_keys(a, t);
    const int n = lead(r, i * 32);
    if (by_row && t < a.T && n == 0)
      for (int k = 0; k < nkv; ++k) ws.desc[t * nkv + k] = make_int4(-1, 0, 0, 0);
    const bool idle = t < a.T && r.keys == 0;
    if (idle && r.pos >= 0) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    for (unsigned todo = __ballot_sync(0xffffffffu, idle); todo; todo &= todo - 1) {
      uint4* o = reinterpret_cast<uint4*>(
          a.out + (size_t)(i * 32 + __ffs(todo) - 1) * a.nq * HD);
      for (int k = lane; k < a.nq * HD / 8; k += 32) o[k] = make_uint4(0, 0, 0, 0);
    }
  }
}

// Parts of one split (group, kv head) added in the order of the keys, a thread
// per four dims of a column and NG parts side by side; each thread requests a
// batch of parts before it uses one.  COL: one column per CTA (few segments of
// many parts), else all columns in a smaller CTA (many segments of a few
// parts, and most CTAs find nothing to do).
constexpr int kJoinThreads = 512;   // at most

template <int HD, bool COL>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const PagedAttnArgs a,
                                                             const PaWork ws, int rpb) {
  constexpr int kJoinBatch = COL ? 8 : 4;
  __shared__ __align__(16) float4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int4 d = ws.desc[blockIdx.x];
  if (d.x < 0) return;
  constexpr int TP = HD / 4;                 // threads per column
  const int G = a.nq / a.kv.n_kv, cols = rpb * G;
  const int width = COL ? TP : cols * TP;    // threads per part
  const int NG = blockDim.x / width;         // parts side by side
  const int tid = threadIdx.x, q = tid / width;
  const int n = COL ? blockIdx.y : tid % width / TP, d4 = tid % TP * 4;
  const int parts = d.y - d.x + 1;
  // part i of the segment: the first CTA's second slot, then first slots
  auto part = [&](int i) { return (size_t)(2 * (d.x + i) + (i == 0 ? 1 : 0)) * cols + n; };
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  bool none = false;
  for (int i0 = 0; i0 < parts && q < NG; i0 += NG * kJoinBatch) {
    float2 ml[kJoinBatch];
    float4 v[kJoinBatch];
    float mx = M;
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j) {
      const int i = i0 + j * NG + q;
      ml[j] = make_float2(-INFINITY, 0.f);
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < parts) {
        ml[j] = ws.ml[part(i)];
        v[j] = *reinterpret_cast<const float4*>(ws.o + part(i) * HD + d4);
      }
    }
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j) {
      none |= ml[j].y == -1.f;               // the group has no such row
      mx = fmaxf(mx, ml[j].x);
    }
    const float ms = mx == -INFINITY ? 0.f : mx;
    const float f0 = exp2_fast(M - ms);
    L *= f0;
    o.x *= f0;
    o.y *= f0;
    o.z *= f0;
    o.w *= f0;
    M = mx;
#pragma unroll
    for (int j = 0; j < kJoinBatch; ++j) {
      const float f = exp2_fast(ml[j].x - ms);
      L += f * ml[j].y;
      o.x += f * v[j].x;
      o.y += f * v[j].y;
      o.z += f * v[j].z;
      o.w += f * v[j].w;
    }
  }
  if (NG > 1) {
    s_ml[tid] = make_float2(M, none ? -1.f : L);
    s_o[tid] = o;
    __syncthreads();
    if (q > 0) return;
    const int ng = min(NG, parts);
    float mx = M;
    for (int i = 1; i < ng; ++i) {
      const float2 ml = s_ml[i * width + tid];
      none |= ml.y == -1.f;
      mx = fmaxf(mx, ml.x);
    }
    const float ms = mx == -INFINITY ? 0.f : mx, f0 = exp2_fast(M - ms);
    L *= f0;
    o.x *= f0;
    o.y *= f0;
    o.z *= f0;
    o.w *= f0;
#pragma unroll 4
    for (int i = 1; i < ng; ++i) {
      const float2 ml = s_ml[i * width + tid];
      const float4 v = s_o[i * width + tid];
      const float f = exp2_fast(ml.x - ms);
      L += ml.y * f;
      o.x += v.x * f;
      o.y += v.y * f;
      o.z += v.z * f;
      o.w += v.w * f;
    }
  }
  if (q > 0 || none) return;
  *reinterpret_cast<uint2*>(a.out + ((size_t)(d.z + n / G) * a.nq + d.w * G + n % G) * HD + d4) =
      make_uint2(pack_bf16(o.x / L, o.y / L), pack_bf16(o.z / L, o.w / L));
}

namespace {

using AttnKernel = void (*)(PagedAttnArgs, PaWork, int, TileWork);

template <bool REST>
AttnKernel attn_kernel(int i) {
  static const AttnKernel k[8] = {
      k_paged_attn<64, false, 1, REST>,  k_paged_attn<64, false, 2, REST>,
      k_paged_attn<64, true, 1, REST>,   k_paged_attn<64, true, 2, REST>,
      k_paged_attn<128, false, 1, REST>, k_paged_attn<128, false, 2, REST>,
      k_paged_attn<128, true, 1, REST>,  k_paged_attn<128, true, 2, REST>};
  return k[i];
}

AttnKernel attn_kernel(int hd, bool e4m3, int nt, bool rest, int* id, size_t* smem) {
  const int rb = hd * (e4m3 ? 1 : 2), i = (hd == 128 ? 4 : 0) + (e4m3 ? 2 : 0) + nt - 1;
  *id = i + (rest ? 8 : 0);
  // the warps' rings and two warps' accumulators
  *smem = (e4m3 ? (size_t)kPaWarps * kPaStages * 2 * 16 * pa_halves(e4m3) * rb : 0) +
          (size_t)kPaWarps / 2 * nt * (hd / 16) * 512;
  return rest ? attn_kernel<true>(i) : attn_kernel<false>(i);
}

constexpr int kPaMaxCtas = 1024;  // CTAs of a launch (workspace size)

// CTAs that fill the current device; 0 on a CUDA error.
int attn_ctas(AttnKernel k, int id, size_t smem) {
  static PerDevice known[16];
  std::atomic<int>& slot = known[id].here();
  int n = slot.load(std::memory_order_relaxed);
  if (!n) {
    int dev = 0, sms = 0, per_sm = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, kPaThreads, smem) != cudaSuccess)
      return 0;
    n = sms * per_sm < kPaMaxCtas ? sms * per_sm : kPaMaxCtas;
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

// Rows that share a group's MMA columns: as many as fit, a power of two.
int attn_rows(int G, int nt) {
  int n = 1;
  while (2 * n * G <= 8 * nt) n *= 2;
  return n;
}

// desc | parts' O | parts' (max, sum), for the largest launch, or the parts of
// the kernel for chunks, which are joined before this one's are written
size_t attn_parts_bytes(int nq, int nkv, int hd) {
  const size_t G = nq / nkv, cols = attn_rows((int)G, 2) * G;
  const size_t n = kPaMaxCtas * (sizeof(int4) + 2 * cols * (hd * sizeof(float) + sizeof(float2)));
  return std::max(n, paged_tile_workspace_bytes(nq, nkv, hd));
}

}  // namespace

// The parts, and the flags between the two kernels.
size_t paged_attn_workspace_bytes(int T, int nq, int nkv, int hd) {
  return T == 0 ? 0 : attn_parts_bytes(nq, nkv, hd) + kTileFlags * sizeof(int32_t);
}

int launch_paged_attn(const PagedAttnArgs& a, bool e4m3, cudaStream_t s, int* launches) {
  const int nkv = a.kv.n_kv, G = a.nq / nkv;
  // Requests with the rows for 48 columns and more on average, and work for the
  // device: the kernel for chunks.  This one -> that: 512 rows, 24/4 heads of 128
  // in bf16, chunks of 8: 215 -> 115 us; 64 rows, 16/2, chunks of 8: 25 -> 22.
  // Not so for 32 columns (512 rows in chunks of 32, 8/8 heads of 64: 42 -> 53)
  // or 256 in all (16 rows, 16/2: 16 -> 21).
  //
  // The average does not say which requests have the rows, so that kernel takes
  // the runs of 32 columns and more and this one what is left of the call (unless
  // there is one request).  63 requests of one row over 4000 keys beside a chunk
  // of 512, 24/4 heads of 128 in bf16: 260 us (88 and 82 by themselves; the blocks
  // of the average's 8 rows fill 48 of 128 columns), 863 by that kernel alone.
  // Calls with nothing left pay for two empty launches: 5 chunks of 64 rows, 8/8
  // heads of 64, e4m3: 19.2 -> 22 us, 8 of 512, 16/2 of 128: 412 -> 417.
  TileWork tile = {};
  const bool chunks = a.req && paged_tile_rows(a) * G >= 48 && (long long)a.T * a.nq >= 1024;
  const bool rest = chunks && a.n_req > 1;
  if (chunks) {
    tile.o = reinterpret_cast<float*>(a.ws);
    tile.left = reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(a.ws) +
                                           attn_parts_bytes(a.nq, nkv, a.kv.hd));
    tile.least = rest ? (31 + G) / G : 0;
    const int rc = launch_paged_tile(a, e4m3, tile, s, launches);
    if (rc) return rc;
    if (!rest) return SLX_OK;
  }
  // Two column tiles where one row needs them, or where a request has the rows
  // to fill them on average and there is work for the device: the keys are read
  // and turned into operands half as often.  One tile -> two, 24/4 heads of 128
  // in bf16: 512 rows in chunks of 4: 290 -> 220 us, of 2: 301 -> 220; 32 rows in
  // chunks of 4: 33 -> 25, 16 rows: 16.6 -> 19.5.  8/8 heads of 64, e4m3, 512
  // rows in chunks of 8 (half a tile): 45 -> 62, of 16: 43 -> 38; 64 rows: 15.3
  // -> 17.1.
  const int tall = attn_rows(G, 2);
  const bool many = !rest && a.req && tall > attn_rows(G, 1) && a.T / tall >= a.n_req &&
                    (long long)a.T * a.nq >= 768;
  const int nt = G > 8 || many ? 2 : 1;
  int id;
  size_t smem;
  const AttnKernel k = attn_kernel(a.kv.hd, e4m3, nt, rest, &id, &smem);
  const int full = attn_ctas(k, id, smem);
  if (full < 1) return SLX_ERR_CUDA;
  // no more CTAs than steps (a unit per warp) the rows could fill
  const long long segs = (long long)a.T * nkv;
  int grid = full;
  if (segs < (long long)full * kPaWarps) {
    const int ku = 16 * pa_halves(e4m3);
    const long long row_units = ((long long)a.max_pages * a.kv.page_size + ku - 1) / ku;
    const long long steps = (segs * row_units + kPaWarps - 1) / kPaWarps;
    if (steps < full) grid = (int)steps;
  }
  const int rpb = a.req ? attn_rows(G, nt) : 1, cols = rpb * G;
  PaWork ws;
  uint8_t* p = reinterpret_cast<uint8_t*>(a.ws);
  ws.desc = reinterpret_cast<int4*>(p);
  ws.o = reinterpret_cast<float*>(p + kPaMaxCtas * sizeof(int4));
  ws.ml = reinterpret_cast<float2*>(ws.o + (size_t)kPaMaxCtas * 2 * cols * a.kv.hd);
  if ((rest ? launch_chained(k, dim3(grid), dim3(kPaThreads), smem, s, a, ws, rpb, tile)
            : launch_k(k, dim3(grid), dim3(kPaThreads), smem, s, a, ws, rpb, tile)) != cudaSuccess)
    return SLX_ERR_CUDA;
  ++*launches;
  // one CTA per column while they fit the device about twice over
  const unsigned n = (unsigned)(segs <= grid ? segs : grid);
  const bool col = n * (unsigned)cols <= 1024;
  auto j = a.kv.hd == 128 ? (col ? k_paged_join<128, true> : k_paged_join<128, false>)
                          : (col ? k_paged_join<64, true> : k_paged_join<64, false>);
  const int width = cols * (a.kv.hd / 4);
  const int threads = col || 2 * width > kJoinThreads ? kJoinThreads : 2 * width;
  if (launch_chained(j, dim3(n, col ? cols : 1), dim3(threads), 0, s, a, ws, rpb) != cudaSuccess)
    return SLX_ERR_CUDA;
  ++*launches;
  return SLX_OK;
}

}  // namespace slx
