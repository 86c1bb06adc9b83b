// Attention of prompt chunks over a paged key-value cache (sm_100a): many rows
// of a request at a time, on the 5th-generation tensor cores.
#include <algorithm>

#include "slx_paged.cuh"
#include "slx_tc.cuh"

namespace slx {

// A CTA takes 128 columns, the (row, q head) pairs of one kv head and of as
// many rows as fit, over 64 keys at a time:
//   S [128 x 64] = Q K^T,   O [128 x hd] += P V     (tcgen05.mma, M = 128)
// with S (twice) and O in TMEM.  A column's lane holds it alone, so maximum and
// sum need no exchange.  P takes the place of its scores in TMEM, the second
// product's first operand, as two 16-bit parts, hi + lo, both multiplied, with
// the bits that they have in the kernel for single tokens.  For bf16 pages O is
// scaled only when a column's maximum has grown by 2^8 (P and the sum stay far
// inside bf16's and fp32's range until then); for e4m3 pages whenever it grows,
// because P takes all of fp16's range (8/8 heads of 64, 512 rows in chunks of 64,
// this kernel alone: 37 us; 34 with 2^8 of the range left for growth, where weights
// below 2^-32 are lost).
// K and V lie in shared memory as their pages have them, rows of
// 64 dims swizzled over 128 bytes: K-major for S, and for P V with the dims
// inside (the descriptor's other order), so neither is transposed.  E4m3 keys
// and values become fp16 on the way (exact), q a power of two times fp16.
//
// Warps 0-3: a column each, S -> P, O.  Warps 4, 5 keys and 6, 7 values: global
// memory to registers a tile ahead, then to one of two places; apart, because
// the fence before the MMAs waits for the loads in flight of its thread.  The
// first thread of each pair issues its MMAs.  Two CTAs per SM (97 KB each), the
// keys of a block of rows cut into parts while that leaves the device unfilled;
// the join adds them in order.
//
// Bound by the chain of the warps that bring the keys: 2800 cycles a tile (loads
// issued 1100, stores and fence 450, the pair's barrier 600, eight MMAs 500;
// the softmax takes 1900), 2400 with two CTAs on an SM; in e4m3 the conversion
// is in it, too, and O is scaled more often.  4096 rows in chunks of 512 over 4k
// to 8k keys, 16/2 heads of 128, in a graph: 417 us in bf16 (about 465 TFLOP/s
// without P's second part), 514 in e4m3, 5 us of each for the kernel behind this
// one; 2214 by the kernel for single tokens.  P through shared memory and one place
// for K and V: 475; values transposed on the way to a K-major operand: 843.
constexpr int kTileM = 128;       // columns (row, q head): the MMAs' M
constexpr int kTileKeys = 64;     // keys per tile
constexpr int kTileThreads = 256;
constexpr int kTileTmem = 256;    // S twice, O
constexpr int kTileCtas = 296;    // two per SM
constexpr int kTileSplits = 8;    // parts of a row at most
// A column's maximum may grow by 2^kTileSlack before O is scaled; P and its sum
// are 2^kTileUp times the softmax's (the quotient is not).
template <bool E4M3>
constexpr float kTileSlack = E4M3 ? 0.f : 8.f;
template <bool E4M3>
constexpr float kTileUp = E4M3 ? 15.f : 0.f;

// Bits of the block's rows, in four words: the first one set at `from` or
// behind it (kTileM: none).
SLX_DEV int next_bit(const uint32_t* m, int from) {
  for (int i = from >> 5; i < kTileM / 32; ++i) {
    uint32_t b = m[i];
    if (i == from >> 5) b &= 0xffffffffu << (from & 31);
    if (b) return 32 * i + __ffs(b) - 1;
  }
  return kTileM;
}

template <int HD, bool E4M3>
__global__ void __launch_bounds__(kTileThreads, 2)
    k_paged_tile(const PagedAttnArgs a, const TileWork ws) {
  constexpr int ES = E4M3 ? 1 : 2, RB = HD * ES;  // bytes of an element, of a key
  constexpr int QB = HD / 64 * kTileM * 128;      // Q: chunks of 64 dims, swizzled
  constexpr int KB = HD / 64 * kTileKeys * 128;   // K likewise
  constexpr int VB = KB;                          // V likewise
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_q, bar_done;
  // by the tile's parity: a warp that runs a tile ahead meets the other barrier
  __shared__ __align__(8) uint64_t bar_k[2], bar_v[2], bar_s[2], bar_p[2], bar_o[2];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ int s_keys[kTileM], s_req[kTileM];
  __shared__ uint32_t s_start[kTileM / 32], s_stop[kTileM / 32];
  __shared__ int s_left[kTileM / 32];
  __shared__ int s_odd[kTileM][2];  // by group's first row: keys with odd values
  uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sQ = base, *sK = sQ + QB, *sV = sK + 2 * KB;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rpb = ws.rpb, nsplit = ws.nsplit;
  const int nkv = a.kv.n_kv, G = a.nq / nkv, ps = a.kv.page_size, sh = a.kv.page_shift;
  const int split = blockIdx.x % nsplit, item = blockIdx.x / nsplit;
  const int kh = item % nkv, row0 = item / nkv * rpb;
  if (tid == 0) {
    mbar_init(&bar_q, 128);
    mbar_init(&bar_done, 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_k[i], 64);
      mbar_init(&bar_v[i], 64);
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], 128);
      mbar_init(&bar_o[i], 1);
    }
    s_abort = 0;
    fence_mbar_init();
  }
  pdl_wait_primary();
  // (TMEM behind the wait, and the next kernel's CTAs let in behind it: one of
  // them that held some while it waits for this kernel could stop it)
  if (warp == 4) {
    tc_alloc(&s_tmem, kTileTmem);
    tc_relinquish();
  }
  // the block's rows, and where its groups (rows of one request) begin and end;
  // with the other kernel behind this one, rows of short runs and idle ones are
  // left to it
  if (tid < kTileM) {
    const RowKeys r = row_keys(a, tid < rpb ? row0 + tid : a.T);
    const bool mine = !ws.least || in_run(a, row0 + 32 * warp, ws.least);
    s_keys[tid] = mine ? r.keys : 0;
    s_req[tid] = r.req;
    s_odd[tid][0] = 0x7fffffff;
    s_odd[tid][1] = -1;
    if (!ws.least && split == 0 && kh == 0 && r.keys == 0 && r.pos >= 0 && tid < rpb)
      set_status(a.status, SLX_ERR_OUT_OF_RANGE);
    s_left[warp] = __any_sync(0xffffffffu, tid < rpb && row0 + tid < a.T && s_keys[tid] == 0);
  }
  __syncthreads();
  if (tid < kTileM) {
    const bool on = s_keys[tid] > 0;
    const bool first = on && (tid == 0 || s_keys[tid - 1] == 0 || s_req[tid - 1] != s_req[tid]);
    const uint32_t st = __ballot_sync(0xffffffffu, first);
    const uint32_t of = __ballot_sync(0xffffffffu, !on || first);
    if (lane == 0) {
      s_start[warp] = st;
      s_stop[warp] = of;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  if (tid == 0 && split == 0 && kh == 0 && ws.n_left)
    ws.left[row0 / rpb] = s_left[0] | s_left[1] | s_left[2] | s_left[3];
  const uint32_t tmem = s_tmem;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_wait(bar, parity & 1, a.status) && !s_abort) return true;
    s_abort = 1;
    return false;
  };
  // the group whose first row is at `from` or behind it, and this split's tiles
  struct Group {
    int r0, r1, req, keys, common, t0, t1;
  };
  auto next_group = [&](int from, Group& p) {
    p.r0 = next_bit(s_start, from);
    if (p.r0 >= kTileM) return false;
    p.r1 = next_bit(s_stop, p.r0 + 1);
    p.req = s_req[p.r0];
    int most = 0, least = 0x7fffffff;
    for (int i = p.r0 + lane; i < p.r1; i += 32) {
      most = max(most, s_keys[i]);
      least = min(least, s_keys[i]);
    }
    p.keys = __reduce_max_sync(0xffffffffu, most);
    p.common = __reduce_min_sync(0xffffffffu, least);
    const int n = (p.keys + kTileKeys - 1) / kTileKeys, per = (n + nsplit - 1) / nsplit;
    p.t0 = min(split * per, n);
    p.t1 = min(p.t0 + per, n);
    return true;
  };
  Group gr;
  int it = 0;  // tiles so far
  const size_t page_bytes = (size_t)2 * nkv * ps * RB, v_off = (size_t)nkv * ps * RB;

  if (warp < 4) {
    // ------------------------------------------------ softmax, a column each --
    const int ri = tid / G, hh = kh * G + tid % G;
    const uint32_t t_lane = tmem + ((uint32_t)(32 * warp) << 16), t_o = t_lane + 2 * kTileKeys;
    if (!ws.least && split == 0 && ri < rpb && row0 + ri < a.T && s_keys[ri] == 0) {
      uint4* o = reinterpret_cast<uint4*>(a.out + ((size_t)(row0 + ri) * a.nq + hh) * HD);
      for (int i = 0; i < HD / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
    }
    bool ok = true;
    for (int from = 0; ok && next_group(from, gr); from = gr.r1) {
      const bool on = ri >= gr.r0 && ri < gr.r1;
      const int lim = on ? s_keys[ri] : 0;
      float m = -INFINITY, l = 0.f;
      if (gr.t1 > gr.t0) {
        // the column's query, swizzled; e4m3 pages: fp16, times a power of two
        // that puts its largest element at 2^12 .. 2^13
        const uint4* qp = reinterpret_cast<const uint4*>(
            a.q + (size_t)(row0 + (on ? ri : gr.r0)) * a.q_stride + (size_t)hh * HD);
        float fac = a.scale * 1.4426950408889634f;
        float up = 1.f;
        if constexpr (E4M3) {
          float mx = 0.f;
          if (on) {
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
              const uint4 v = qp[i];
              const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(x[j])), fabsf(bf16_hi(x[j]))));
            }
          }
          const int e = (int)(__float_as_uint(mx) >> 23) - 127;
          const int k = mx == 0.f || e == 128 ? 0 : min(12 - e, 100);
          up = __uint_as_float((uint32_t)(127 + k) << 23);
          fac *= a.kv.k_scale[kh] * __uint_as_float((uint32_t)(127 - k) << 23);
        }
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          uint4 v = on ? qp[i] : make_uint4(0, 0, 0, 0);
          if constexpr (E4M3) {
            uint32_t* x = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = pack_f16x2(bf16_lo(x[j]) * up, bf16_hi(x[j]) * up);
          }
          *reinterpret_cast<uint4*>(sQ + (i >> 3) * (kTileM * 128) + tid * 128 +
                                    (((i & 7) ^ (tid & 7)) << 4)) = v;
        }
        fence_proxy_async();
        mbar_arrive(&bar_q);
        for (int t = gr.t0; t < gr.t1; ++t, ++it) {
          const int k0 = t * kTileKeys, b = it & 1;
          ok = __all_sync(0xffffffffu, wait(&bar_s[b], it >> 1));
          if (!ok) break;
          tc_fence_after();
          uint32_t r[4][16];
#pragma unroll
          for (int i = 0; i < 4; ++i) tc_ld16(t_lane + b * kTileKeys + 16 * i, r[i]);
          tc_wait_ld();
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              float s = __uint_as_float(r[i][j]) * fac;
              if (k0 + kTileKeys > gr.common && k0 + 16 * i + j >= lim) s = -INFINITY;
              r[i][j] = __float_as_uint(s);
              mx = fmaxf(mx, s);
            }
          const bool more = mx > m + kTileSlack<E4M3>;
          const float top = more ? mx : m, ms = top == -INFINITY ? 0.f : top;
          const float f = more ? exp2_fast(m - ms) : 1.f, mt = ms - kTileUp<E4M3>;
          m = top;
          l *= f;
          if (t > gr.t0 && __any_sync(0xffffffffu, more)) {
            // (the products with the tile before are done)
            ok = __all_sync(0xffffffffu, wait(&bar_o[1 - b], (it - 1) >> 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < HD / 16; ++i) {
              uint32_t o[16];
              tc_ld16(t_o + 16 * i, o);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tc_st16(t_o + 16 * i, o);
            }
            tc_wait_st();
          }
          // P takes the scores' place: 32 columns of high parts, 32 of low ones
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float p0 = exp2_fast(__uint_as_float(r[i][2 * j]) - mt);
              const float p1 = exp2_fast(__uint_as_float(r[i][2 * j + 1]) - mt);
              l += p0 + p1;
              if constexpr (!E4M3) {
                hi[j] = pack_bf16(p0, p1);
                lo[j] = pack_bf16(p0 - bf16_lo(hi[j]), p1 - bf16_hi(hi[j]));
              } else {
                hi[j] = pack_f16x2(p0, p1);
                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
                lo[j] = pack_f16x2(p0 - h.x, p1 - h.y);
              }
            }
            tc_st8(t_lane + b * kTileKeys + 8 * i, hi);
            tc_st8(t_lane + b * kTileKeys + kTileKeys / 2 + 8 * i, lo);
          }
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(&bar_p[b]);
        }
        ok = ok && __all_sync(0xffffffffu, wait(&bar_o[(it - 1) & 1], (it - 1) >> 1));
        if (!ok) break;
        tc_fence_after();
      }
      // O / l, or this split's part of it
      const float sv = E4M3 ? a.kv.v_scale[kh] : 1.f;
      const float scale = nsplit == 1 ? sv / l : sv;
      const size_t part = (size_t)blockIdx.x * (rpb * G) + tid;
      const volatile int* odd = s_odd[gr.r0];
      const int odd0 = odd[0], odd1 = min(odd[1], lim - 1);
      if (nsplit > 1 && on) ws.ml[part] = make_float2(m, l);
#pragma unroll 1
      for (int i = 0; gr.t1 > gr.t0 && i < HD / 16; ++i) {
        uint32_t r[16];
        __syncwarp();
        tc_ld16(t_o + 16 * i, r);
        tc_wait_ld();
        if (!on) continue;
        float o[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = __uint_as_float(r[j]) * scale;
        // infinite and NaN values that some rows do not attend were left out
        for (int k = odd0; k <= odd1; ++k) {
          const int page = a.table[(size_t)gr.req * a.max_pages + (k >> sh)];
          if ((unsigned)page >= (unsigned)a.kv.n_pages) continue;
          const uint8_t* v = a.kv.base + (size_t)page * page_bytes + v_off +
                             ((size_t)kh * ps + (k & (ps - 1))) * RB + 16 * i * ES;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x;
            if constexpr (E4M3)
              x = (v[j] & 0x7f) == 0x7f ? __uint_as_float(0x7fc00000u) : 0.f;
            else
              x = bf16_to_f32(reinterpret_cast<const uint16_t*>(v)[j]);
            if (!(fabsf(x) < INFINITY)) o[j] += x;
          }
        }
        if (nsplit == 1) {
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = pack_bf16(o[2 * j], o[2 * j + 1]);
          uint4* d = reinterpret_cast<uint4*>(a.out + ((size_t)(row0 + ri) * a.nq + hh) * HD +
                                              16 * i);
          d[0] = make_uint4(w[0], w[1], w[2], w[3]);
          d[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
          float4* d = reinterpret_cast<float4*>(ws.o + part * HD + 16 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            d[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
      }
    }
  } else {
    // ----------------------- keys (warps 4, 5) and values (warps 6, 7): global
    // memory -> registers, a tile ahead, -> operands.  (Apart: the fence before
    // the MMAs waits for a thread's loads too.)
    const int t = tid & 63;
    const size_t kh_off = (size_t)kh * ps * RB;
    // where the tile's four runs of 16 keys lie, by lane (-1: nowhere; what is
    // loaded in their place, and behind the group's keys, is cleared when the
    // tile is stored: `held` has a bit for each run)
    auto page_at = [&](int tile) {
      const int k = tile * kTileKeys + 16 * (lane & 3);
      return tile < gr.t1 && k < gr.keys ? a.table[(size_t)gr.req * a.max_pages + (k >> sh)] : -2;
    };
    auto run_at = [&](int tile, int p) -> long long {
      const int k = tile * kTileKeys + 16 * (lane & 3);
      if ((unsigned)p < (unsigned)a.kv.n_pages)
        return (long long)((size_t)(unsigned)p * page_bytes + kh_off + (k & (ps - 1)) * RB);
      if (tile < gr.t1 && k < gr.keys) set_status(a.status, SLX_ERR_OUT_OF_RANGE);
      return -1;
    };
    constexpr int PK = RB / 16, KK = 64 / PK;  // 16-byte pieces of a key, keys of a pass
    const bool is_v = warp >= 6;
    const uint8_t* src = a.kv.base + (is_v ? v_off : 0) + t / PK * RB + t % PK * 16;
    uint8_t* dst = is_v ? sV : sK;     // two tiles
    uint4 kr[PK];
    unsigned held = 0;
    auto fetch = [&](int tile, int page) {
      const long long run = run_at(tile, page);
      held = __ballot_sync(0xffffffffu, run >= 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* p = src + __shfl_sync(0xffffffffu, max(run, 0LL), i);
#pragma unroll
        for (int j = 0; j < 16 / KK; ++j)
          kr[i * 16 / KK + j] = __ldg(reinterpret_cast<const uint4*>(p + j * KK * RB));
      }
    };
    // what the operand holds of them: 16-bit elements
    constexpr int PW = E4M3 ? 2 : 1;
    uint4 op[E4M3 ? PK : 1][2];
    auto prepare = [&](int k0) {
      if (k0 + kTileKeys > gr.keys || (held & 15) != 15) {
#pragma unroll
        for (int j = 0; j < PK; ++j)
          if (k0 + j * KK + t / PK >= gr.keys || !(held >> j * KK / 16 & 1))
            kr[j] = make_uint4(0, 0, 0, 0);
      }
      if (is_v && k0 + kTileKeys > gr.common) {
        // a weight of 0 does not hide an infinite or NaN value from the rows
        // that do not attend its key
#pragma unroll
        for (int j = 0; j < PK; ++j) {
          uint32_t x[4] = {kr[j].x, kr[j].y, kr[j].z, kr[j].w};
          bool odd = false;
          // (elements of 16 or 8 bits; `e` is a value's exponent, all ones)
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int h = 0; h < 4 / ES; ++h) {
              const uint32_t e = (E4M3 ? 0x7fu : 0x7f80u) << 8 * ES * h;
              if ((x[w] & e) == e) {
                x[w] &= ~((E4M3 ? 0xffu : 0xffffu) << 8 * ES * h);
                odd = true;
              }
            }
          if (!odd) continue;
          kr[j] = make_uint4(x[0], x[1], x[2], x[3]);
          atomicMin(&s_odd[gr.r0][0], k0 + j * KK + t / PK);
          atomicMax(&s_odd[gr.r0][1], k0 + j * KK + t / PK);
        }
      }
      if constexpr (E4M3) {
#pragma unroll
        for (int j = 0; j < PK; ++j) {
          e4m3x4(kr[j].x, op[j][0].x, op[j][0].y);
          e4m3x4(kr[j].y, op[j][0].z, op[j][0].w);
          e4m3x4(kr[j].z, op[j][1].x, op[j][1].y);
          e4m3x4(kr[j].w, op[j][1].z, op[j][1].w);
        }
      }
    };
    auto store = [&](int b) {
#pragma unroll
      for (int j = 0; j < PK; ++j)
#pragma unroll
        for (int h = 0; h < PW; ++h) {
          const int key = j * KK + t / PK, p = t % PK * PW + h;
          uint8_t* at = dst + b * KB + (p >> 3) * (kTileKeys * 128) + key * 128;
          *reinterpret_cast<uint4*>(at + (((p & 7) ^ (key & 7)) << 4)) =
              E4M3 ? op[E4M3 ? j : 0][h] : kr[j];
        }
    };
    const uint64_t q_desc = sdesc_sw128(smem_u32(sQ)), k_desc = sdesc_sw128(smem_u32(sK));
    const uint64_t v_desc = sdesc_sw128_mn(smem_u32(sV), kTileKeys * 128);
    bool ok = true;
    int grp = 0;  // groups with tiles
    for (int from = 0; ok && next_group(from, gr); from = gr.r1) {
      if (gr.t1 == gr.t0) continue;
      fetch(gr.t0, page_at(gr.t0));
      int page = page_at(gr.t0 + 1);
      for (int tl = gr.t0; tl < gr.t1; ++tl, ++it) {
        prepare(tl * kTileKeys);
        // K's place is free when the tile two before has its scores, V's when it
        // is multiplied
        const int b = it & 1;
        ok = __all_sync(0xffffffffu,
                        it < 2 || wait(is_v ? &bar_o[b] : &bar_s[b], (it >> 1) - 1));
        if (!ok) break;
        store(b);
        fence_proxy_async();
        mbar_arrive(is_v ? &bar_v[b] : &bar_k[b]);
        if (is_v) {
          if (tl + 1 < gr.t1) fetch(tl + 1, page);
          page = page_at(tl + 2);
          if (t == 0 && wait(&bar_p[b], it >> 1) && wait(&bar_v[b], it >> 1)) {
            tc_fence_after();
            // (descriptors count in 16 bytes)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc_mma_ts(tmem + 2 * kTileKeys, tmem + b * kTileKeys + h * (kTileKeys / 2) + 8 * k,
                          v_desc + b * (VB / 16) + 128 * k,
                          (E4M3 ? idesc_f16(HD) : idesc_bf16(HD)) | kIdescBmn,
                          tl > gr.t0 || (h | k) != 0);
            tc_commit(&bar_o[b]);
          }
        } else {
          // (one thread for all of them: it meets every group's bar_q in turn)
          if (t == 0 && (tl > gr.t0 || wait(&bar_q, grp)) && wait(&bar_k[b], it >> 1) &&
              (it < 2 || wait(&bar_o[b], (it >> 1) - 1))) {
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc_mma_ss(tmem + b * kTileKeys, q_desc + c * (kTileM * 8) + 2 * k,
                          k_desc + b * (KB / 16) + c * (kTileKeys * 8) + 2 * k,
                          E4M3 ? idesc_f16(kTileKeys) : idesc_bf16(kTileKeys), (c | k) != 0);
            tc_commit(&bar_s[b]);
          }
          __syncwarp();
          if (tl + 1 < gr.t1) fetch(tl + 1, page);
          page = page_at(tl + 2);
        }
        __syncwarp();
      }
      ++grp;
    }
  }
  if (tid == 128 || tid == 192) {  // the threads that issue the MMAs
    tc_commit(&bar_done);
    mbar_wait(&bar_done, 0, a.status);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tc_dealloc(tmem, kTileTmem);
  }
}

// A warp per (row, q head): its splits' parts in the order of the keys.
template <int HD>
__global__ void __launch_bounds__(256) k_paged_tile_join(const PagedAttnArgs a, const TileWork ws) {
  pdl_launch_dependents();
  pdl_wait_primary();
  const int lane = threadIdx.x & 31, rpb = ws.rpb, nsplit = ws.nsplit;
  const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (id >= (long long)a.T * a.nq) return;
  const int row = (int)(id / a.nq), hh = (int)(id % a.nq), G = a.nq / a.kv.n_kv;
  const int col = row % rpb * G + hh % G;
  const size_t item = (size_t)(row / rpb) * a.kv.n_kv + hh / G;
  auto part = [&](int i) { return (item * nsplit + i) * (rpb * G) + col; };
  // (requested with the row; of no use where the row has no parts)
  const float2 ml = lane < nsplit ? ws.ml[part(lane)] : make_float2(-INFINITY, 0.f);
  const RowKeys r = row_keys(a, row);
  const bool mine = !ws.least || in_run(a, row, ws.least);  // (lane 0: this row)
  if (r.keys == 0 || !__shfl_sync(0xffffffffu, mine, 0)) return;
  float4 v[4], o = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool on = lane < HD / 4;
  float M = ml.x;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const float ms = M == -INFINITY ? 0.f : M, f = exp2_fast(ml.x - ms);
  float L = ml.y * f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
  for (int i0 = 0; i0 < nsplit; i0 += 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      // (a split without tiles has written no O)
      const float sum = __shfl_sync(0xffffffffu, ml.y, (i0 + j) & 31);
      if (on && i0 + j < nsplit && sum != 0.f)
        v[j] = *reinterpret_cast<const float4*>(ws.o + part(i0 + j) * HD + 4 * lane);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float g = __shfl_sync(0xffffffffu, f, (i0 + j) & 31);
      o.x += v[j].x * g;
      o.y += v[j].y * g;
      o.z += v[j].z * g;
      o.w += v[j].w * g;
    }
  }
  if (on)
    *reinterpret_cast<uint2*>(a.out + ((size_t)row * a.nq + hh) * HD + 4 * lane) =
        make_uint2(pack_bf16(o.x / L, o.y / L), pack_bf16(o.z / L, o.w / L));
}

size_t paged_tile_workspace_bytes(int nq, int nkv, int hd) {
  const size_t G = nq / nkv, cols = kTileM / G * G;
  return kTileCtas * cols * (hd * sizeof(float) + sizeof(float2));
}

// Rows of a block: as many as fit, or as a request has on average (a block
// with the rows of several takes them one after the other).
int paged_tile_rows(const PagedAttnArgs& a) {
  const int most = kTileM / (a.nq / a.kv.n_kv), each = a.T / a.n_req;
  return each < most ? (each > 0 ? each : 1) : most;
}

// Lays out the parts behind ws.o, fills in how the rows are cut, and joins them.
int launch_paged_tile(const PagedAttnArgs& a, bool e4m3, TileWork& ws, cudaStream_t s,
                      int* launches) {
  const int nkv = a.kv.n_kv, G = a.nq / nkv, hd = a.kv.hd, rpb = paged_tile_rows(a);
  const int cols = rpb * G, blocks = (a.T + rpb - 1) / rpb;
  const long long items = (long long)blocks * nkv;
  if (items > 0x7fffffff / kTileSplits) return SLX_ERR_UNSUPPORTED;
  // splits of four tiles and more in the longest request up to two CTAs per SM,
  // of two up to one (64 rows over 600 keys, 24/4 heads: 20 -> 17 us; 320 rows over
  // 200 to 1500, 8/8, has the four: 19 by this kernel alone, by two 21)
  const long long tiles = ((long long)a.max_pages * a.kv.page_size + kTileKeys - 1) / kTileKeys;
  auto splits = [&](int ctas, int least) {
    const long long n = std::min(ctas / items, tiles / least);
    return (int)std::max(1LL, std::min(n, (long long)kTileSplits));
  };
  const int nsplit = std::max(splits(kTileCtas, 4), splits(kTileCtas / 2, 2));
  ws.ml = reinterpret_cast<float2*>(ws.o + (size_t)items * nsplit * cols * hd);
  ws.rpb = rpb;
  ws.nsplit = nsplit;
  ws.n_left = ws.least && blocks <= kTileFlags ? blocks : 0;
  using Kernel = void (*)(PagedAttnArgs, TileWork);
  const Kernel k = hd == 128 ? (e4m3 ? k_paged_tile<128, true> : k_paged_tile<128, false>)
                             : (e4m3 ? k_paged_tile<64, true> : k_paged_tile<64, false>);
  // Q, two tiles of K and of V, and what aligns them
  const size_t smem = (size_t)hd / 64 * (kTileM + 4 * kTileKeys) * 128 + 1024;
  static PerDevice configured[4];
  std::atomic<int>& slot = configured[(hd == 128 ? 2 : 0) + e4m3].here();
  if (!slot.load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess)
      return SLX_ERR_CUDA;
    slot.store(1, std::memory_order_relaxed);
  }
  if (launch_k(k, dim3((unsigned)(items * nsplit)), dim3(kTileThreads), smem, s, a, ws) !=
      cudaSuccess)
    return SLX_ERR_CUDA;
  ++*launches;
  if (nsplit == 1) return SLX_OK;
  const long long warps = (long long)a.T * a.nq;
  if (launch_chained(hd == 128 ? k_paged_tile_join<128> : k_paged_tile_join<64>,
                     dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, s, a, ws) != cudaSuccess)
    return SLX_ERR_CUDA;
  ++*launches;
  return SLX_OK;
}

}  // namespace slx
