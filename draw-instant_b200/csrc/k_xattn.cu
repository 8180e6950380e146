// k_xattn.cu — attention over an encoder's states, with lengths and a key mask per request (sm_100a).
//
//   O[b,i,h] = sum_j softmax_j(scale Q[b,i,h] . K[b,j,g]) V[b,j,g],  g = h / (H / Hkv),
//   over the valid keys j < min(kv_len[b], Skv) with key_mask[b][j] != 0
//
// A request without valid keys gives zero rows; query rows from q_len[b] on are not written.
//
// One pass over the keys with a running maximum and sum per row.  Query heads that share a key head are
// packed as rows of one tile (row t = token * GP + head, GP the power of two in the group), so a
// key tile is read once for all of them and single-token queries fill rows that would be padding.  A work unit is 256
// packed rows of one (request, head group) and a range of 128-key tiles; one persistent CTA per SM walks its units:
//
//   warps 0-3, 4-7  softmax of rows 0..127 and 128..255, one row per thread (= one TMEM lane)
//   warp 8          MMA issue: S = Q K^T into TMEM, O += P V with P read from TMEM
//   warp 9          TMA loads: Q tiles of the next unit while this one runs, K and V tiles through one ring
//
// P (16-bit) overwrites the columns of the scores it came from; the two row tiles alternate on the tensor
// pipe, so one tile's products run while the other's exponentials do.  MMAs of the one issuing thread
// execute in order: S of tile j + 1 may follow P V of tile j into the same columns, and its commit also tells that
// P V of tile j is complete.  The running maximum only moves when a row's true maximum passes it by 2^8, so O is rarely
// rescaled and P stays below 2^8 in range of both types; O / l is exact under the stale maximum.
// P is rounded to the inputs' 16-bit type for the second product (half a step per probability, averaged over the
// keys); scores, maxima, sums and O are 32-bit.
//
// Masked keys: scores become -inf before the maximum, and the V rows of masked keys are zeroed in shared memory before
// the product, so nothing they hold reaches O.
// Few units: the key tiles of a unit are split over CTAs, each writing (O, max, sum) in 32 bits to the
// workspace, and a second kernel joins them in split order.
#include <algorithm>
#include <cstring>

#include "di_common.cuh"

namespace di {

struct XattnParams {
  CUtensorMap tmQ, tmK, tmV;
  void* O;
  long long osb, oss, osh;  // output strides in elements
  int kvb_mul, kvh_mul, vb_mul, vh_mul, qb_mul, qh_mul;  // 0: the tensor is expanded over that axis
  int B, HG, GP, gps, G;    // head groups of GP = 2^gps query heads; G query heads per key head
  int Sq, Skv, RT, NS;      // row tiles (256 rows) per group, key splits
  int nq, ring;             // Q buffers, K/V ring tiles
  int wide;                 // output rows take 32-byte stores
  const int *q_len, *kv_len;
  const unsigned char* mask;
  float scale_log2;
  float* part;              // [NS][B * HG * R][D] partial O, then [NS][B * HG * R][2] (max, sum)
  int* err;
};

namespace {

constexpr int QT = 128, KT = 128;
constexpr int kXThreads = 384;
// Registers: three warpgroups launch with 168 each; the softmax warpgroups (a row of 128 scores per thread) take
// 216, the third gives up its own down to 64: 256 * 216 + 128 * 64 <= 384 * 168.
constexpr float kRescale = 8.0f;  // log2 units

template <int D>
struct XSmem {
  static constexpr uint32_t TILE = 128 * D * 2;       // one Q, K or V tile
  static constexpr uint32_t HALF = 128 * 128;         // 64 columns of it, 128-byte rows
  static constexpr int SLOTS = D == 64 ? 13 : 7;
  static constexpr int MAXRING = SLOTS - 2;
  static constexpr uint32_t TOTAL = 1024 + SLOTS * TILE + 1024;
};

__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float lo_f(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_f(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float ex2_approx(float x) {  // 2^x; -inf -> +0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2,
                                            int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, "
      "%7}], [%2];" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1),
      "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc]: A's 16-bit values lie two to a column, row m in lane m
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Position in a ring of n buffers: entry e lies in buffer e % n and completes its barrier's phase (e / n) & 1.
struct RingPos {
  int s = 0, ph = 0;
  __device__ __forceinline__ void advance(int n, int by = 1) {
    s += by;
    if (s >= n) { s -= n; ph ^= 1; }
  }
  __device__ __forceinline__ RingPos next(int n) const {
    RingPos r = *this;
    r.advance(n);
    return r;
  }
};

// One work unit: packed rows [row0, row0 + rows) of (b, hg), key tiles [t0, t1) of n valid-range keys.
struct Unit {
  int b, hg, sp, row0, rows, n, t0, t1;
};
__device__ __forceinline__ bool unit_of(const XattnParams& p, unsigned u, Unit& w) {
  w.sp = (int)(u % p.NS);
  u /= p.NS;
  const int rt = (int)(u % p.RT);
  u /= p.RT;
  w.hg = (int)(u % p.HG);
  w.b = (int)(u / p.HG);
  w.row0 = rt * 2 * QT;
  const int q = p.q_len ? min(max(__ldg(p.q_len + w.b), 0), p.Sq) : p.Sq;
  w.rows = min(q * p.GP - w.row0, 2 * QT);
  w.n = p.kv_len ? min(max(__ldg(p.kv_len + w.b), 0), p.Skv) : p.Skv;
  const int nt = (w.n + KT - 1) / KT;
  w.t0 = (int)((long long)nt * w.sp / p.NS);
  w.t1 = (int)((long long)nt * (w.sp + 1) / p.NS);
  return w.rows > 0;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(kXThreads, 1) xattn_kernel(const __grid_constant__ XattnParams p) {
  using S = XSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                             // [nq][2] tiles
  uint8_t* sKV = smem + p.nq * 2 * S::TILE;       // [ring] tiles
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::SLOTS * S::TILE);
  uint64_t* q_full = bars;                        // [2]
  uint64_t* q_empty = bars + 2;                   // [2]
  uint64_t* kv_full = bars + 4;                   // [ring]
  uint64_t* kv_empty = kv_full + S::MAXRING;      // [ring]
  uint64_t* s_full = kv_empty + S::MAXRING;       // [2] scores of row tile w ready
  uint64_t* p_full = s_full + 2;                  // [2] probabilities of row tile w written
  uint64_t* o_full = p_full + 2;                  // [2] O of row tile w complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < p.ring; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();
  const unsigned units = (unsigned)p.B * p.HG * p.RT * p.NS;
  // TMEM columns: scores of row tile w at 128 w (its probabilities over their first half), O at 256 + D w

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == 9) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tmQ);
      tma_prefetch_desc(&p.tmK);
      tma_prefetch_desc(&p.tmV);
      RingPos kv, q;
      unsigned nkv = 0, nq = 0;  // copies issued, up to the buffers there are
      for (unsigned u = blockIdx.x; u < units && !*abort_flag; u += gridDim.x) {
        Unit w;
        if (!unit_of(p, u, w) || w.t0 >= w.t1) continue;
        const int nw = w.rows > QT ? 2 : 1;
        if (!mbar_wait(&q_empty[q.s], q.ph ^ 1, p.err, DEVERR_WAIT_TMA)) { *abort_flag = 1; break; }
        mbar_arrive_expect_tx(&q_full[q.s], nw * S::TILE);
        for (int i = 0; i < nw; ++i)
          for (int c = 0; c < D / 64; ++c)
            tma_load_5d(sQ + (q.s * 2 + i) * S::TILE + c * S::HALF, &p.tmQ, &q_full[q.s], c * 64, 0,
                        (w.row0 + i * QT) >> p.gps, w.hg * p.qh_mul, w.b * p.qb_mul);
        q.advance(p.nq);
        ++nq;
        const int hk = w.hg * p.GP / p.G;
        for (int t = w.t0; t < w.t1; ++t)
          for (int v = 0; v < 2; ++v) {
            if (*abort_flag || !mbar_wait(&kv_empty[kv.s], kv.ph ^ 1, p.err, DEVERR_WAIT_TMA)) {
              *abort_flag = 1;
              t = w.t1;
              break;
            }
            mbar_arrive_expect_tx(&kv_full[kv.s], S::TILE);
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(sKV + kv.s * S::TILE + c * S::HALF, v ? &p.tmV : &p.tmK, &kv_full[kv.s], c * 64, t * KT,
                          hk * (v ? p.vh_mul : p.kvh_mul), w.b * (v ? p.vb_mul : p.kvb_mul));
            kv.advance(p.ring);
            ++nkv;
          }
      }
      if (*abort_flag) {  // leave no copy in flight behind: the last ones issued into each buffer
        for (unsigned i = 0; i < min(nkv, (unsigned)p.ring); ++i) {
          kv.s = kv.s ? kv.s - 1 : (kv.ph ^= 1, p.ring - 1);
          mbar_wait(&kv_full[kv.s], kv.ph, p.err, DEVERR_WAIT_TMA);
        }
        for (unsigned i = 0; i < min(nq, (unsigned)p.nq); ++i) {
          q.s = q.s ? q.s - 1 : (q.ph ^= 1, p.nq - 1);
          mbar_wait(&q_full[q.s], q.ph, p.err, DEVERR_WAIT_TMA);
        }
      }
    }
  } else if (warp == 8) {
    if (elect_one()) {
      RingPos kv, q;
      bool ok = true;
      int ph_p[2] = {0, 0};
      for (unsigned u = blockIdx.x; ok && u < units; u += gridDim.x) {
        Unit w;
        if (!unit_of(p, u, w) || w.t0 >= w.t1) continue;
        const int nw = w.rows > QT ? 2 : 1, qb = q.s;
        ok = !*abort_flag && mbar_wait(&q_full[q.s], q.ph, p.err, DEVERR_WAIT_MMA);
        q.advance(p.nq);
        auto kv_wait = [&](const RingPos& r) {
          return !*abort_flag && mbar_wait(&kv_full[r.s], r.ph, p.err, DEVERR_WAIT_MMA);
        };
        auto keys16 = [&](int t) { return (min(w.n - t * KT, KT) + 15) / 16; };  // 16-key steps of tile t
        auto issue_s = [&](int i, int t, int slot) {
          const uint32_t aQ = smem_u32(sQ + (qb * 2 + i) * S::TILE), aK = smem_u32(sKV + slot * S::TILE);
          // the score tile is as wide as the softmax reads it: 32-key chunks
          const uint32_t id = idesc_f16(128, 0, BF16) | ((uint32_t)(((keys16(t) + 1) / 2 * 32) >> 3) << 17);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * S::HALF + (kk % 4) * 32;
            umma_f16(tmem + i * 128, sdesc_sw128(aQ + off, 16, 1024), sdesc_sw128(aK + off, 16, 1024), id, kk != 0);
          }
          umma_commit(&s_full[i]);
        };
        auto issue_pv = [&](int i, int t, int slot) {
          const uint32_t aV = smem_u32(sKV + slot * S::TILE);
          constexpr uint32_t id = idesc_f16(128, D, BF16, false, true);  // V is MN-major (d contiguous)
          const int steps = keys16(t);
          for (int kk = 0; kk < steps; ++kk)
            umma_f16_ta(tmem + 256 + i * D, tmem + i * 128 + kk * 8, sdesc_sw128(aV + kk * 2048, S::HALF, 1024), id,
                        t != w.t0 || kk != 0);
        };
        if (ok && (ok = kv_wait(kv))) {
          tc_fence_after();
          for (int i = 0; i < nw; ++i) issue_s(i, w.t0, kv.s);
          umma_commit(&kv_empty[kv.s]);
        }
        for (int t = w.t0; ok && t < w.t1; ++t) {  // kv: the K tile of t, then its V tile, then the next K tile
          const bool more = t + 1 < w.t1;
          const RingPos v = kv.next(p.ring), k2 = v.next(p.ring);
          ok = kv_wait(v) && (!more || kv_wait(k2));
          for (int i = 0; ok && i < nw; ++i) {
            ok = !*abort_flag && mbar_wait(&p_full[i], ph_p[i], p.err, DEVERR_WAIT_MMA);
            ph_p[i] ^= 1;
            if (!ok) break;
            tc_fence_after();
            issue_pv(i, t, v.s);
            if (more) issue_s(i, t + 1, k2.s);
            else umma_commit(&o_full[i]);
          }
          if (!ok) break;
          umma_commit(&kv_empty[v.s]);
          if (more) umma_commit(&kv_empty[k2.s]);
          else umma_commit(&q_empty[qb]);
          kv = k2;
        }
      }
      if (!ok) *abort_flag = 1;
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- softmax warps: one packed row per thread ----------------
    const int i = warp / 4, wq = warp & 3;
    const int lrow = wq * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tmem + i * 128 + lane_off, tO = tmem + 256 + i * D + lane_off;
    const long long R = (long long)p.Sq * p.GP;
    int ph_s = 0, ph_o = 0;
    RingPos v;  // the V tile of the current key tile (first row tile's warps only: every unit has that one)
    v.advance(p.ring);
    bool ok = true;
    for (unsigned u = blockIdx.x; ok && u < units; u += gridDim.x) {
      Unit w;
      if (!unit_of(p, u, w)) continue;
      const int row = i * QT + lrow;               // row of the unit
      const bool mine = row < w.rows;
      const bool warp_on = i * QT + wq * 32 < w.rows;
      float m_run = -INFINITY, l_run = 0.f;
      if (i * QT < w.rows) {
        for (int t = w.t0; ok && t < w.t1; ++t) {
          ok = !*abort_flag && mbar_wait(&s_full[i], ph_s, p.err, DEVERR_WAIT_SOFTMAX);
          ok = __all_sync(0xffffffffu, ok);
          ph_s ^= 1;
          if (!ok) break;
          tc_fence_after();
          const int left = w.n - t * KT;  // > 0; keys of this tile inside the length
          const int nc = min(4, (left + 31) / 32);
          uint32_t bits[4];
          const bool partial = left < KT || p.mask;
          if (partial) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int j = t * KT + c * 32 + lane;
              bits[c] = __ballot_sync(0xffffffffu, j < w.n && (!p.mask || __ldg(p.mask + (long long)w.b * p.Skv + j)));
            }
            // V rows of masked keys inside the tensor are zeroed (one key per thread of the first row tile; keys
            // past Skv are zero already)
            if (i == 0) {
              ok = mbar_wait(&kv_full[v.s], v.ph, p.err, DEVERR_WAIT_SOFTMAX);
              const uint32_t mine_bits = wq == 0 ? bits[0] : wq == 1 ? bits[1] : wq == 2 ? bits[2] : bits[3];
              if (ok && !((mine_bits >> lane) & 1) && lrow < (left + 15) / 16 * 16) {
                uint8_t* vrow = sKV + v.s * S::TILE + lrow * 128;
#pragma unroll
                for (int c = 0; c < D / 8; ++c)
                  *reinterpret_cast<uint4*>(vrow + (c / 8) * S::HALF + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
                fence_async_smem();
              }
              __syncwarp();
            }
          }
          if (warp_on) {
            float s[KT];
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (c < nc) tmem_ld32(tS + c * 32, reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
            tmem_wait_ld();
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (c < nc) {
                if (partial && bits[c] != 0xffffffffu) {
#pragma unroll
                  for (int k = 0; k < 32; ++k)
                    if (!((bits[c] >> k) & 1)) s[c * 32 + k] = -INFINITY;
                }
                float a = -INFINITY, b = -INFINITY;
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                  a = max3f(a, s[c * 32 + k], s[c * 32 + k + 1]);
                  b = max3f(b, s[c * 32 + k + 2], s[c * 32 + k + 3]);
                }
                mx = max3f(mx, a, b);
              }
            mx *= p.scale_log2;  // the scale is positive
            const bool move = mx > m_run + kRescale;
            const float m_new = move ? mx : m_run;
            const float alpha = move ? ex2_approx(m_run - m_new) : 1.0f;
            const float m_sub = m_new == -INFINITY ? 0.f : m_new;  // no valid key yet: every p is 2^-inf = 0
            const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), nm2 = f2_pack(-m_sub, -m_sub);
            uint64_t acc2 = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (c < nc) {
                uint32_t pk[16];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                  const uint64_t x = fma2(f2_pack(s[c * 32 + k], s[c * 32 + k + 1]), sc2, nm2);
                  const float a = ex2_approx(lo_f(x)), b = ex2_approx(hi_f(x));
                  acc2 = add2(acc2, f2_pack(a, b));
                  pk[k / 2] = pack2<BF16>(a, b);
                }
                tmem_st16(tS + c * 16, pk);
              }
            l_run = l_run * alpha + (lo_f(acc2) + hi_f(acc2));
            m_run = m_new;
            if (t != w.t0 && __any_sync(0xffffffffu, move)) {
              // this tile's scores follow the previous P V on the tensor pipe: O is complete
#pragma unroll
              for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld32(tO + c * 32, r);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
                tmem_st32(tO + c * 32, r);
              }
            }
            tmem_wait_st();
          }
          tc_fence_before();
          mbar_arrive(&p_full[i]);
          v.advance(p.ring, 2);
        }
        if (ok && w.t1 > w.t0) {
          ok = !*abort_flag && mbar_wait(&o_full[i], ph_o, p.err, DEVERR_WAIT_SOFTMAX);
          ok = __all_sync(0xffffffffu, ok);
          ph_o ^= 1;
          tc_fence_after();
        }
        if (ok && warp_on) {
          const long long tr = w.row0 + row;  // packed row of the group
          const long long pr = ((long long)w.b * p.HG + w.hg) * R + tr + (long long)w.sp * p.B * p.HG * R;
          const bool any = w.t1 > w.t0;
          const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
          uint16_t* o = static_cast<uint16_t*>(p.O) + w.b * p.osb + (tr >> p.gps) * p.oss +
                        (w.hg * p.GP + (tr & (p.GP - 1))) * p.osh;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            if (any) {  // warp-uniform
              tmem_ld32(tO + c * 32, r);
              tmem_wait_ld();
            }
            if (p.NS > 1) {
              if (mine && any) {
                float4* d = reinterpret_cast<float4*>(p.part + pr * D + c * 32);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  d[k] = make_float4(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1]),
                                     __uint_as_float(r[4 * k + 2]), __uint_as_float(r[4 * k + 3]));
              }
            } else if (mine) {
              uint32_t h[16];
#pragma unroll
              for (int k = 0; k < 16; ++k)  // no valid key: zeros, whatever O holds
                h[k] = l_run == 0.f ? 0u : pack2<BF16>(__uint_as_float(r[2 * k]) * inv, __uint_as_float(r[2 * k + 1]) * inv);
              if (p.wide) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
                  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(o + c * 32 + k * 16),
                               "r"(h[8 * k]), "r"(h[8 * k + 1]), "r"(h[8 * k + 2]), "r"(h[8 * k + 3]), "r"(h[8 * k + 4]),
                               "r"(h[8 * k + 5]), "r"(h[8 * k + 6]), "r"(h[8 * k + 7])
                               : "memory");
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  reinterpret_cast<uint4*>(o + c * 32)[k] = make_uint4(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
              }
            }
          }
          if (p.NS > 1 && mine)
            reinterpret_cast<float2*>(p.part + (long long)p.NS * p.B * p.HG * R * D)[pr] = make_float2(m_run, l_run);
        }
        tc_fence_before();  // O is read before the next unit's first P V, which waits for this warp's p_full
      }
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the key splits: one warp per packed row.
template <bool BF16, int D>
__global__ void __launch_bounds__(128) xattn_join_kernel(const __grid_constant__ XattnParams p) {
  pdl_begin();
  const long long R = (long long)p.Sq * p.GP, NR = (long long)p.B * p.HG * R;
  const long long r = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (r >= NR) return;
  const int b = (int)(r / R / p.HG), hg = (int)(r / R % p.HG);
  const long long t = r % R;
  if (p.q_len && t / p.GP >= __ldg(p.q_len + b)) return;
  const float2* ml = reinterpret_cast<const float2*>(p.part + p.NS * NR * D);
  float m = -INFINITY;
  for (int s = lane; s < p.NS; s += 32) {
    const float2 v = ml[s * NR + r];
    if (v.y != 0.f) m = fmaxf(m, v.x);
  }
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  constexpr int W = D / 32;
  float acc[W] = {}, l = 0.f;
  for (int s = 0; s < p.NS; ++s) {
    const float2 v = ml[s * NR + r];
    if (v.y == 0.f) continue;  // nothing valid in this split (its O may not even be written); NaN passes
    const float f = ex2_approx(v.x - m);
    l = fmaf(v.y, f, l);
    const float* o = p.part + (s * NR + r) * D + lane * W;
#pragma unroll
    for (int k = 0; k < W; ++k) acc[k] = fmaf(o[k], f, acc[k]);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t* o = static_cast<uint16_t*>(p.O) + b * p.osb + t / p.GP * p.oss + (hg * p.GP + t % p.GP) * p.osh + lane * W;
#pragma unroll
  for (int k = 0; k < W; k += 2) reinterpret_cast<uint32_t*>(o)[k / 2] = pack2<BF16>(acc[k] * inv, acc[k + 1] * inv);
}

struct XPlan {
  int GP, HG, RT, NS;
};
XPlan xattn_plan(const Ctx* c, int B, int H, int Hkv, int Sq, int Skv) {
  XPlan x;
  const int G = H / Hkv;
  x.GP = G & -G;  // packed heads: the power of two in the group (tiles of 128 rows hold whole tokens)
  if (x.GP > QT) x.GP = QT;
  x.HG = H / x.GP;
  x.RT = (int)(((long long)Sq * x.GP + 2 * QT - 1) / (2 * QT));
  const long long units = (long long)B * x.HG * x.RT;
  const int nt = (Skv + KT - 1) / KT;
  x.NS = 1;
  if (units * 2 <= c->num_sms) x.NS = (int)std::max<long long>(1, std::min<long long>(nt, 2 * c->num_sms / units));
  return x;
}

template <bool BF16, int D>
int launch_xattn(Ctx* c, XattnParams& p, int nt) {
  using S = XSmem<D>;
  auto kern = xattn_kernel<BF16, D>;
  static unsigned attr_done = 0;
  if (!(attr_done & (1u << (c->device & 31)))) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::TOTAL) != cudaSuccess)
      return set_error(c, DI_ECUDA, "cross_attention: shared memory attribute");
    attr_done |= 1u << (c->device & 31);
  }
  p.nq = D == 64 || nt <= 2 ? 2 : 1;
  p.ring = S::SLOTS - 2 * p.nq;
  const long long units = (long long)p.B * p.HG * p.RT * p.NS;
  launch_k(kern, dim3((unsigned)std::min<long long>(units, c->num_sms)), kXThreads, S::TOTAL, c->stream, p);
  if (p.NS > 1) {
    const int rc = check_launch(c, "cross_attention");
    if (rc != DI_OK) return rc;
    const long long rows = (long long)p.B * p.HG * p.Sq * p.GP;
    launch_k(xattn_join_kernel<BF16, D>, dim3((unsigned)((rows + 3) / 4)), 128, 0, c->stream, p);
  }
  return check_launch(c, "cross_attention");
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" size_t di_cross_attention_workspace(di_ctx_t h, int B, int H, int Hkv, int Sq, int Skv, int D) {
  if (!h || B <= 0 || H <= 0 || Hkv <= 0 || Sq <= 0 || Skv <= 0 || D <= 0 || H % Hkv) return 0;
  const XPlan x = xattn_plan(ctx_of(h), B, H, Hkv, Sq, Skv);
  return x.NS > 1 ? (size_t)x.NS * B * H * Sq * (D + 2) * 4 : 0;
}

extern "C" int di_cross_attention(di_ctx_t h, int dtype, const void* Q, const long long q_strides[3], const void* K,
                                  const long long k_strides[3], const void* V, const long long v_strides[3], void* O,
                                  const long long o_strides[3], int B, int H, int Hkv, int Sq, int Skv, int D,
                                  const int* q_len, const int* kv_len, const unsigned char* key_mask, float scale,
                                  void* ws, size_t ws_bytes) {
  Ctx* c = ctx_of(h);
  if (!c || (dtype != DI_F16 && dtype != DI_BF16)) return DI_EINVAL;
  DeviceGuard guard(c->device);
  if (B <= 0 || H <= 0 || Hkv <= 0 || Sq <= 0 || Skv <= 0 || !Q || !K || !V || !O || !q_strides || !k_strides ||
      !v_strides || !o_strides)
    return set_error(c, DI_EINVAL, "cross_attention: bad shape or missing tensor");
  if (H % Hkv) return set_error(c, DI_EINVAL, "cross_attention: H must be a multiple of Hkv");
  if (D != 64 && D != 128) return set_error(c, DI_EUNSUPPORTED, "cross_attention: head dim must be 64 or 128");
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(O))
    return set_error(c, DI_EINVAL, "cross_attention: pointers must be 16-byte aligned");
  const XPlan x = xattn_plan(c, B, H, Hkv, Sq, Skv);
  if ((long long)Sq * x.GP > (1 << 30) || Skv > (1 << 30) || (long long)B * x.HG * x.RT * x.NS > 0x7fffffffll)
    return set_error(c, DI_EUNSUPPORTED, "cross_attention: too many tokens");
  // strides of axes of length one mean nothing: they are replaced by 8 elements (a valid tensor-map stride)
  long long qs[3], ks[3], vs[3], os[3];
  for (int i = 0; i < 3; ++i) {
    const int nq = i == 0 ? B : i == 1 ? Sq : H, nk = i == 0 ? B : i == 1 ? Skv : Hkv;
    qs[i] = nq > 1 ? q_strides[i] : 8;
    ks[i] = nk > 1 ? k_strides[i] : 8;
    vs[i] = nk > 1 ? v_strides[i] : 8;
    os[i] = nq > 1 ? o_strides[i] : 16;
    if (qs[i] < 0 || ks[i] < 0 || vs[i] < 0 || (qs[i] | ks[i] | vs[i] | os[i]) % 8 || os[i] < 0)
      return set_error(c, DI_EINVAL, "cross_attention: strides must be multiples of 8 elements and not negative");
    if (os[i] == 0) return set_error(c, DI_EINVAL, "cross_attention: the output's rows must not share memory");
  }
  if (qs[1] == 0 || ks[1] == 0 || vs[1] == 0 || (qs[2] == 0 && x.GP > 1))
    return set_error(c, DI_EINVAL, "cross_attention: tokens and grouped query heads cannot be expanded");
  if (!(scale > 0.f) || !(scale < INFINITY)) return set_error(c, DI_EINVAL, "cross_attention: scale must be positive and finite");
  const size_t need = di_cross_attention_workspace(h, B, H, Hkv, Sq, Skv, D);
  if (need && (!ws || ws_bytes < need || !aligned16(ws)))
    return set_error(c, DI_EINVAL, "cross_attention: workspace missing, too small or not 16-byte aligned");
  XattnParams p;
  memset(&p, 0, sizeof p);
  const CUtensorMapDataType dt = dtype == DI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  std::string err;
  // an expanded axis (stride 0) becomes an axis of length one whose coordinate stays 0
  auto len = [](long long stride, int n) { return (uint64_t)(stride ? n : 1); };
  auto str = [](long long stride) { return (uint64_t)(stride ? stride : 8) * 2; };
  const uint64_t qd[5] = {(uint64_t)D, (uint64_t)x.GP, (uint64_t)Sq, len(qs[2], x.HG), len(qs[0], B)};
  const uint64_t qst[4] = {str(qs[2]), str(qs[1]), str(qs[2] * x.GP), str(qs[0])};
  const uint32_t qbox[5] = {64, (uint32_t)x.GP, (uint32_t)(QT / x.GP), 1, 1};
  const uint32_t kbox[4] = {64, KT, 1, 1};
  const uint64_t kd[4] = {(uint64_t)D, (uint64_t)Skv, len(ks[2], Hkv), len(ks[0], B)};
  const uint64_t vd[4] = {(uint64_t)D, (uint64_t)Skv, len(vs[2], Hkv), len(vs[0], B)};
  const uint64_t kst[3] = {str(ks[1]), str(ks[2]), str(ks[0])}, vst[3] = {str(vs[1]), str(vs[2]), str(vs[0])};
  if (!make_tmap(&p.tmQ, dt, 5, Q, qd, qst, qbox, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmK, dt, 4, K, kd, kst, kbox, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmV, dt, 4, V, vd, vst, kbox, CU_TENSOR_MAP_SWIZZLE_128B, &err))
    return set_error(c, DI_EINVAL, "cross_attention: " + err);
  p.qh_mul = qs[2] != 0; p.qb_mul = qs[0] != 0;
  p.kvh_mul = ks[2] != 0; p.kvb_mul = ks[0] != 0;
  p.vh_mul = vs[2] != 0; p.vb_mul = vs[0] != 0;
  p.O = O;
  p.osb = os[0]; p.oss = os[1]; p.osh = os[2];
  p.wide = (reinterpret_cast<uintptr_t>(O) & 31) == 0 && (os[0] | os[1] | os[2]) % 16 == 0;
  while ((1 << p.gps) < x.GP) ++p.gps;
  p.B = B; p.HG = x.HG; p.GP = x.GP; p.G = H / Hkv; p.Sq = Sq; p.Skv = Skv; p.RT = x.RT; p.NS = x.NS;
  p.q_len = q_len; p.kv_len = kv_len; p.mask = key_mask;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(ws);
  p.err = c->d_err;
  const int nt = (Skv + KT - 1) / KT;
  if (dtype == DI_F16) return D == 64 ? launch_xattn<false, 64>(c, p, nt) : launch_xattn<false, 128>(c, p, nt);
  return D == 64 ? launch_xattn<true, 64>(c, p, nt) : launch_xattn<true, 128>(c, p, nt);
}
