// What the attention kernels over paged caches share.
#pragma once
#include "slx_kernels.cuh"

namespace slx {

SLX_DEV uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

SLX_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// four e4m3 bytes -> two fp16 pairs (exact; NaN stays NaN)
SLX_DEV void e4m3x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 t, u; mov.b32 {t, u}, %2; cvt.rn.f16x2.e4m3x2 %0, t; "
      "cvt.rn.f16x2.e4m3x2 %1, u;}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}

// Row t's request and the keys it attends: pos + 1, 0 for an idle row or one
// out of range.  (Both are read at once: rows are read in batches.)
struct RowKeys {
  int req, pos, keys;
};
SLX_DEV RowKeys row_keys(const PagedAttnArgs& a, int t) {
  RowKeys r = {0, -1, 0};
  if (t < a.T) {
    r.pos = a.pos[t];
    r.req = a.req ? a.req[t] : t;
  }
  const bool ok = (unsigned)r.req < (unsigned)a.n_req &&
                  (unsigned)r.pos >> a.kv.page_shift < (unsigned)a.max_pages && r.pos >= 0;
  r.keys = ok ? r.pos + 1 : 0;
  return r;
}

// For a warp over rows t0 .. t0 + 31: whether row t0 + lane stands in a run of
// `least` rows or more (at most 32) that name the same request.  The rows before
// and behind the 32 are looked at, so every kernel of a call has the same answer.
SLX_DEV bool in_run(const PagedAttnArgs& a, int t0, int least) {
  const int lane = threadIdx.x & 31;
  int r[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int t = t0 + 32 * (i - 1) + lane;
    r[i] = t >= 0 && t < a.T ? a.req[t] : 0;
  }
  uint32_t same[3];  // as the row before
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int t = t0 + 32 * (i - 1) + lane;
    int before = __shfl_up_sync(0xffffffffu, r[i], 1);
    const int last = i ? __shfl_sync(0xffffffffu, r[i ? i - 1 : 0], 31) : 0;
    if (lane == 0) before = last;
    same[i] = __ballot_sync(0xffffffffu, before == r[i] && t > 0 && t < a.T && i + lane > 0);
  }
  const uint64_t left = ((uint64_t)same[1] << 32 | same[0]) << (31 - lane);
  const uint64_t right = ((uint64_t)same[2] << 32 | same[1]) >> (lane + 1);
  return t0 + lane < a.T && __clzll(~left) + __ffsll(~right) >= least;
}

// Workspace of k_paged_tile, and how a call's rows are cut for it.
struct TileWork {
  int32_t* left;  // [n_left] whether a block has rows for the kernel behind it
  float* o;       // [items][splits][cols][hd]
  float2* ml;     // [items][splits][cols] max (log2), sum
  int n_left;     // (0: no flags)
  int least;      // rows of the runs that it takes (0: it takes all rows)
  int rpb, nsplit;
};

}  // namespace slx
