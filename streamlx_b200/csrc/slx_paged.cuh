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

}  // namespace slx
