// k_xattn.cu — attention over an encoder's states, with lengths and a key mask per request (sm_100a).
//
//   O[b,i,h] = sum_j softmax_j(scale Q[b,i,h] . K[b,j,g]) V[b,j,g],  g = h / (H / Hkv),
//   over the valid keys j < min(kv_len[b], Skv) with key_mask[b][j] != 0
//
// A request without valid keys gives zero rows; query rows from q_len[b] on are not written.
//
// One pass over the keys with a running maximum and sum per row.  Query heads that share a key head are
// packed as rows (row t = token * GP + head, GP the power of two in the group), so a key tile is read once for all of
// them and single-token queries fill rows that would be padding.  One persistent CTA per SM:
//
//   4 NW warps  softmax: NW groups of 128 rows, one row per thread (= one TMEM lane)
//   MMA warp    S = Q K^T into TMEM, O += P V with P read from TMEM
//   TMA warp    Q tiles of the next work item while this one runs, K and V tiles through one ring
//   clean warp  zeroes the V rows of masked keys in shared memory (their P is 0, but 0 * inf is not)
//   item warp   works out the items ahead of the others and hands them over through shared memory
//
// P (16-bit) overwrites the columns of scores that have been read.  The groups take turns on the tensor pipe, so one
// group's products run while the others' exponentials do.  MMAs of the one issuing thread execute in order: S of the next
// key tile may follow P V into the same columns, and its commit also tells that P V is complete.  The running maximum
// only moves when a row's true maximum passes it by 2^8, so O is rarely rescaled and P stays below 2^8, in range of both
// types; O / l is exact under the stale maximum.  Scores, maxima, sums and O are 32-bit.  P is rounded to the inputs' 16-bit
// type for the second product, half a step per probability: the roundings of a row's keys are independent, but O shrinks
// with the number of keys as they do, so O carries the error of one more rounding beside its own, up to 1.4 times the
// error of a result that is rounded once (measured against 64 bits, bf16 2.3e-3 and 1.7e-3, fp16 2.7e-4 and 2.1e-4).  A second
// 16-bit part of P would remove it for a second P V, half as many MMAs again.
//
// Work, by rows: an item is up to NW tiles of 128 rows of one (request, head group), which share its key tiles.
// Work, by keys (too few rows for the SMs): an item is a range of key tiles of one tile of rows; the key tiles of all
// requests are laid end to end and cut into as many equal ranges as there are CTAs, whatever the lengths, and the
// groups of a CTA take its key tiles in turn.  Each group writes (O, max, sum) in 32 bits to the workspace and a second
// kernel joins them in key order.
//
// Key tiles are 128 keys.  Two groups (TMEM holds 128 columns of S and D of O for each); at head dim 64 with up to 128
// keys three, whose O lies over the spent scores: an item is then one tile of keys, and S of the next item's group i is
// issued behind P V of this item's group i + 1.
//
// O of a warp whose 32 rows are all to be written goes through shared memory (the group's Q tile, which is spent) and a TMA
// store; ragged rows are stored from registers.
//
// Bound and measured (graph replays).  Long, 2 x 8 heads (4 of keys), 4096 queries, 8191 keys, head dim 128, bf16: 241 us,
// 1050 TFLOP/s (16 heads, 8 of keys, of 64: 428 us).  A key tile of both groups takes 3600 cycles, of which the MMAs need 2048 and the exponentials as many;
// the rest is each group's chain of score wait, maximum, exponentials and P V, and 256 items on 148 SMs make two rounds
// of 1.73.  Short, 16 x 5 heads, 4096 queries, 77 keys, head dim 64, fp16: 26.0 us, 3.3 TB/s, the same chain once per item.
// By keys, 16 x 16 heads (4 of keys), one query, 8192 keys: 39.8 us, 4.1 TB/s, six of them the second kernel's.
#include <algorithm>
#include <cstring>

#include "di_common.cuh"

namespace di {

struct XattnParams {
  CUtensorMap tmQ, tmK, tmV, tmO;
  void* O;
  long long osb, oss, osh;  // output strides in elements
  int kb_mul, kh_mul, vb_mul, vh_mul, qb_mul, qh_mul;  // 0: the tensor is expanded over that axis
  int B, HG, GP, gps, G;    // head groups of GP = 2^gps query heads; G query heads per key head
  int Sq, Skv, RT, tpi;     // row blocks per group, row tiles per item
  int by_keys;
  unsigned items;           // by rows: B * HG * RT
  int d_rt, d_hg, d_b;      // gridDim.x in units of the item order (b, hg, rt)
  int nq, ring;             // Q buffers, K/V ring tiles
  int wide;                 // output rows take 32-byte stores
  const int *q_len, *kv_len;
  const unsigned char* mask;
  float scale_log2;
  float* part;              // by keys: [slots][NW][128][D] partial O, then [slots][NW][128][2] (max, sum)
  int slots, grid;
  int* err;
};

namespace {

constexpr float kRescale = 8.0f;  // log2 units
constexpr int KT = 128;          // keys per tile
constexpr int kQBufs = 3;         // most Q buffers
constexpr int kItems = 4;         // work items worked out ahead
constexpr int kMaxByKeys = 256;   // requests whose key tiles are laid end to end

template <int D, bool SHORT>
struct XCfg {
  static constexpr int NW = SHORT ? 3 : 2;                      // groups of 128 rows
  static constexpr int NH = SHORT ? 1 : 2, KS = KT / NH;        // P of a tile is handed over in NH parts of KS keys
  static constexpr int SW = 4 * NW;                             // softmax warps
  static constexpr int THREADS = 32 * SW + 128;
  static constexpr int TCOLS = SHORT ? 128 : 256;                    // TMEM columns of a group: S (P over it), O
  static constexpr int TO = SHORT ? 64 : 128;                   // first column of O
  static constexpr uint32_t TILE = 128 * D * 2, HALF = 128 * 128;  // Q, K or V tile; 64 columns of it (128-byte rows)
  static constexpr uint32_t DATA = D == 64 ? 13 * 16384 : 7 * 32768;
  static constexpr int MAXRING = 10;
  static constexpr uint32_t BARS = 8 * (2 * kQBufs * NW + 3 * MAXRING + NW * NH + 3 * NW + 2 * kItems) + 16 + kItems * 64;
  static constexpr uint32_t TOTAL = 1024 + DATA + (BARS + 15) / 16 * 16 + (kMaxByKeys + 4) * 4;
  static_assert(TOTAL <= 232448, "shared memory of one CTA");
  // Registers a lane once the roles have shared them out (two groups): the scores of a whole row stay in them.
  static constexpr int SOFT_REGS = 216, SERVICE_REGS = 72;
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
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
// Waits for tcgen05.ld; the registers it fills pass through, so that nothing reads them before.
__device__ __forceinline__ void wait_ld(float (&s)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(s[0]), "+f"(s[1]), "+f"(s[2]), "+f"(s[3]), "+f"(s[4]), "+f"(s[5]), "+f"(s[6]), "+f"(s[7]),
                 "+f"(s[8]), "+f"(s[9]), "+f"(s[10]), "+f"(s[11]), "+f"(s[12]), "+f"(s[13]), "+f"(s[14]), "+f"(s[15]),
                 "+f"(s[16]), "+f"(s[17]), "+f"(s[18]), "+f"(s[19]), "+f"(s[20]), "+f"(s[21]), "+f"(s[22]), "+f"(s[23]),
                 "+f"(s[24]), "+f"(s[25]), "+f"(s[26]), "+f"(s[27]), "+f"(s[28]), "+f"(s[29]), "+f"(s[30]), "+f"(s[31])
               ::"memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
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
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tma_store_5d(const CUtensorMap* m, const void* src, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
               : "memory");
}
// Gives back something that was only read: nothing is published, so no release (which would wait for earlier stores).
__device__ __forceinline__ void mbar_arrive_relaxed(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
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
__device__ __forceinline__ uint64_t kdesc(uint32_t a) { return sdesc_sw128(0, 16, 1024) | (a >> 4); }  // K-major tile

// Bounded wait that also ends when another role has given up; the flag is read only when the phase is not there yet.
__device__ __forceinline__ bool wait_on(uint64_t* bar, int ph, volatile int* abort_flag, int* err, int code) {
  if (mbar_try_wait(smem_u32(bar), ph)) return true;
  return !*abort_flag && mbar_wait(bar, ph, err, code);
}

// Position in a ring of n buffers: entry e lies in buffer e % n and completes its barrier's phase (e / n) & 1.
struct RingPos {
  int s = 0, ph = 0;
  __device__ __forceinline__ void advance(int n) {
    if (++s == n) { s = 0; ph ^= 1; }
  }
  __device__ __forceinline__ RingPos next(int n) const {
    RingPos r = *this;
    r.advance(n);
    return r;
  }
  __device__ __forceinline__ void back(int n) {
    if (--s < 0) { s = n - 1; ph ^= 1; }
  }
};

// A work item: packed rows [row0, row0 + rows) of (b, hg), key tiles [t0, t1) of its n keys in reach.
struct Item {
  int b, hg, row0, rows, n, t0, t1, slot;  // rows 0: no more items
};
// The items of one CTA.  Items without rows are left out; those without keys are kept when they are by rows (their
// outputs are zeros).
struct Items {
  const XattnParams& p;
  const int* ends;  // by keys: key tiles of the requests before and with b, times row blocks and head groups
  unsigned u;       // by rows
  int b, hg, rt;
  int g, g1, bb;    // by keys: this CTA's range of the tiles laid end to end, request of tile g
  __device__ __forceinline__ Items(const XattnParams& p_, const int* e) : p(p_), ends(e) {
    if (p.by_keys) {
      const long long total = ends[p.B - 1];
      g = (int)(total * blockIdx.x / p.grid);
      g1 = (int)(total * (blockIdx.x + 1) / p.grid);
      bb = 0;
    } else {
      u = blockIdx.x;
      rt = (int)(u % p.RT);
      hg = (int)(u / p.RT % p.HG);
      b = (int)(u / p.RT / p.HG);
    }
  }
  __device__ __forceinline__ bool next(Item& w) {
    if (p.by_keys) {
      while (g < g1) {
        while (ends[bb] <= g) ++bb;
        w.b = bb;
        w.n = p.kv_len ? min(max(__ldg(p.kv_len + bb), 0), p.Skv) : p.Skv;
        const int nt = (w.n + KT - 1) / KT, at = g - (bb ? ends[bb - 1] : 0);
        const int blk = at / nt;
        w.t0 = at - blk * nt;
        w.t1 = min(nt, w.t0 + g1 - g);
        w.hg = blk / p.RT;
        const int r = blk - w.hg * p.RT;
        w.slot = (int)blockIdx.x + (bb * p.HG + w.hg) * p.RT + r;  // grows by one with each CTA and each block of rows
        g += w.t1 - w.t0;
        if (rows_of(w, r)) return true;
      }
      return false;
    }
    while (u < p.items) {
      w.b = b;
      w.hg = hg;
      const int r = rt;
      u += gridDim.x;
      rt += p.d_rt;
      hg += p.d_hg;
      b += p.d_b;
      if (rt >= p.RT) { rt -= p.RT; ++hg; }
      if (hg >= p.HG) { hg -= p.HG; ++b; }
      if (!rows_of(w, r)) continue;
      w.n = p.kv_len ? min(max(__ldg(p.kv_len + w.b), 0), p.Skv) : p.Skv;
      w.t0 = 0;
      w.t1 = (w.n + KT - 1) / KT;
      w.slot = 0;
      return true;
    }
    return false;
  }
  __device__ __forceinline__ bool rows_of(Item& w, int r) {
    w.row0 = r * p.tpi * 128;
    const int q = p.q_len ? min(max(__ldg(p.q_len + w.b), 0), p.Sq) : p.Sq;
    w.rows = min((q << p.gps) - w.row0, p.tpi * 128);
    return w.rows > 0;
  }
};

template <bool BF16, int D, bool SHORT>
__global__ void __launch_bounds__(XCfg<D, SHORT>::THREADS, 1) xattn_kernel(const __grid_constant__ XattnParams p) {
  using C = XCfg<D, SHORT>;
  constexpr int NW = C::NW, NH = C::NH, KS = C::KS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int qtiles = p.by_keys ? 1 : p.tpi;        // Q tiles of an item
  uint8_t* sQ = smem;                              // [nq][qtiles]
  uint8_t* sKV = smem + p.nq * qtiles * C::TILE;  // [ring]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::DATA);  // [nq][NW] Q tile of group i
  uint64_t* q_empty = q_full + kQBufs * NW;        // [nq][NW]
  uint64_t* kv_full = q_empty + kQBufs * NW;       // [ring]
  uint64_t* kv_empty = kv_full + C::MAXRING;       // [ring] products over, and seen by the clean warp
  uint64_t* v_clean = kv_empty + C::MAXRING;       // [ring] V rows of masked keys zeroed
  uint64_t* s_full = v_clean + C::MAXRING;         // [NW] scores ready
  uint64_t* p_full = s_full + NW;                  // [NW][NH] probabilities written
  uint64_t* o_full = p_full + NW * NH;             // [NW] O complete
  uint64_t* o_read = o_full + NW;                  // [NW] O read (SHORT: the next scores may overwrite it)
  uint64_t* item_full = o_read + NW;               // [kItems]
  uint64_t* item_empty = item_full + kItems;       // [kItems]
  Item* items = reinterpret_cast<Item*>(item_empty + kItems);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(items) + kItems * 64);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* ends = reinterpret_cast<int*>(smem + C::DATA + (C::BARS + 15) / 16 * 16);  // [B] by keys

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int svc = warp - C::SW;  // service warps: 0 MMA, 1 TMA, 2 clean, 3 items
  if (threadIdx.x == 0) {
    for (int i = 0; i < kQBufs * NW; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], p.by_keys ? C::SW : 4); }
    for (int i = 0; i < p.ring; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 2); mbar_init(&v_clean[i], 1); }
    for (int i = 0; i < NW; ++i) {
      mbar_init(&s_full[i], 1);
      for (int h = 0; h < NH; ++h) mbar_init(&p_full[i * NH + h], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_read[i], 4);
    }
    for (int i = 0; i < kItems; ++i) { mbar_init(&item_full[i], 1); mbar_init(&item_empty[i], 3 + C::SW); }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (svc == 0) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  pdl_begin();
  if (p.by_keys && svc == 3) {  // running sums of the requests' key tiles
    int sum = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b < p.B) n = ((p.kv_len ? min(max(__ldg(p.kv_len + b), 0), p.Skv) : p.Skv) + KT - 1) / KT * p.HG * p.RT;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += x;
      }
      if (b < p.B) ends[b] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // a tile needs its V rows cleaned when it has masked keys inside the tensor (rows past Skv are zero already)
  auto cleaned = [&](const Item& w, int t) { return p.mask || (w.n < p.Skv && w.n - t * KT < KT); };
  // The next item, or nothing, for a single thread; done() gives its place back.
  RingPos ip;
  auto taken = [&](bool ok) -> const Item* {
    if (!ok) {
      *abort_flag = 1;
      return nullptr;
    }
    return items[ip.s].rows ? &items[ip.s] : nullptr;
  };
  auto next = [&](int code) { return taken(wait_on(&item_full[ip.s], ip.ph, abort_flag, p.err, code)); };
  // The same for a whole warp: its lanes agree on the wait, as one that left alone would be missing from what follows.
  auto next_all = [&](int code) {
    return taken(__all_sync(0xffffffffu, wait_on(&item_full[ip.s], ip.ph, abort_flag, p.err, code)));
  };
  auto done = [&] {
    mbar_arrive_relaxed(&item_empty[ip.s]);
    ip.advance(kItems);
  };

  if (svc >= 0) {
    if constexpr (!SHORT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::SERVICE_REGS));
    if (svc == 1) {
      if (elect_one()) {
        tma_prefetch_desc(&p.tmQ);
        tma_prefetch_desc(&p.tmK);
        tma_prefetch_desc(&p.tmV);
        RingPos kv, q;
        unsigned nkv = 0;                // copies issued
        unsigned q_used = 0, q_any = 0;  // Q tiles loaded, modulo 2, and at all
        bool ok = true;
        for (const Item* item; ok && (item = next(DEVERR_WAIT_TMA)); done()) {
          const Item w = *item;
          if (w.t0 >= w.t1) continue;
          for (int i = 0; ok && i * 128 < w.rows; ++i) {
            // a group that earlier items left out is behind: its buffer's phase has a count of its own
            const int qi = q.s * NW + i;
            if (!(ok = wait_on(&q_empty[qi], ((q_used >> qi) & 1) ^ 1, abort_flag, p.err, DEVERR_WAIT_TMA))) break;
            q_used ^= 1u << qi;
            q_any |= 1u << qi;
            mbar_arrive_expect_tx(&q_full[qi], C::TILE);
            for (int c = 0; c < D / 64; ++c)
              tma_load_5d(sQ + (q.s * qtiles + i) * C::TILE + c * C::HALF, &p.tmQ, &q_full[qi], c * 64, 0,
                          (w.row0 + i * 128) >> p.gps, w.hg * p.qh_mul, w.b * p.qb_mul);
          }
          q.advance(p.nq);
          const int hk = (w.hg << p.gps) / p.G;
          for (int t = w.t0; ok && t < w.t1; ++t)
            for (int v = 0; v < 2; ++v) {
              if (!(ok = wait_on(&kv_empty[kv.s], kv.ph ^ 1, abort_flag, p.err, DEVERR_WAIT_TMA))) break;
              mbar_arrive_expect_tx(&kv_full[kv.s], C::TILE);
              for (int c = 0; c < D / 64; ++c)
                tma_load_4d(sKV + kv.s * C::TILE + c * C::HALF, v ? &p.tmV : &p.tmK, &kv_full[kv.s], c * 64, t * KT,
                            hk * (v ? p.vh_mul : p.kh_mul), w.b * (v ? p.vb_mul : p.kb_mul));
              kv.advance(p.ring);
              ++nkv;
            }
        }
        if (!ok || *abort_flag) {  // leave no copy in flight behind: the last ones issued into each buffer
          *abort_flag = 1;
          for (unsigned i = 0; i < min(nkv, (unsigned)p.ring); ++i) {
            kv.back(p.ring);
            mbar_wait(&kv_full[kv.s], kv.ph, p.err, DEVERR_WAIT_TMA);
          }
          for (int i = 0; i < kQBufs * NW; ++i)
            if ((q_any >> i) & 1) mbar_wait(&q_full[i], ((q_used >> i) & 1) ^ 1, p.err, DEVERR_WAIT_TMA);
        }
      }
    } else if (svc == 0) {
      if (elect_one()) {
        RingPos kv, q;
        bool ok = true;
        unsigned ph_p = 0, ph_c = 0, ph_r = 0;  // phases of p_full, v_clean, o_read, one bit each
        unsigned used = 0;                      // groups whose O has to be read before new scores (SHORT)
        unsigned ph_q = 0;                      // phases of q_full
        auto wait = [&](uint64_t* b, int ph) { return wait_on(b, ph, abort_flag, p.err, DEVERR_WAIT_MMA); };
        {
          auto issue_s = [&](const Item& w, int i, int qt, int t, int slot) {  // qt: Q tile
            if (SHORT) {
              if ((used >> i) & 1) {
                ok = wait(&o_read[i], (ph_r >> i) & 1);
                ph_r ^= 1u << i;
                tc_fence_after();
              }
              used |= 1u << i;
            }
            const uint64_t dq = kdesc(smem_u32(sQ + qt * C::TILE)), dk = kdesc(smem_u32(sKV + slot * C::TILE));
            // the score tile is as wide as the softmax reads it: 32-key chunks
            const int n = min((w.n - t * KT + 31) / 32, KT / 32) * 32;
            const uint32_t id = idesc_f16(128, 0, BF16) | ((uint32_t)(n >> 3) << 17);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma_f16(tmem + i * C::TCOLS, dq + ((kk / 4) * C::HALF + (kk % 4) * 32) / 16,
                       dk + ((kk / 4) * C::HALF + (kk % 4) * 32) / 16, id, kk != 0);
            umma_commit(&s_full[i]);
          };
          auto issue_pv = [&](const Item& w, int i, int t, int h, int slot, bool first) {  // first: of the item's tiles
            const uint64_t dv = sdesc_sw128(0, C::HALF, 1024) | (smem_u32(sKV + slot * C::TILE + h * KS * 128) >> 4);
            constexpr uint32_t id = idesc_f16(128, D, BF16, false, true);  // V is MN-major (d contiguous)
            const int steps = min((w.n - t * KT - h * KS + 15) / 16, KS / 16);
#pragma unroll
            for (int kk = 0; kk < KS / 16; ++kk)
              if (kk < steps)
                umma_f16_ta(tmem + i * C::TCOLS + C::TO, tmem + i * C::TCOLS + h * (KS / 2) + kk * 8, dv + kk * 2048 / 16, id,
                            !first || h != 0 || kk != 0);
          };
          auto v_wait = [&](const Item& w, const RingPos& v, int t) {
            if (!wait(&kv_full[v.s], v.ph)) return false;
            if (cleaned(w, t)) {
              if (!wait(&v_clean[v.s], (ph_c >> v.s) & 1)) return false;
              ph_c ^= 1u << v.s;
            }
            return true;
          };
          auto p_wait = [&](int i, int h) {
            const bool r = wait(&p_full[i * NH + h], (ph_p >> (i * NH + h)) & 1);
            ph_p ^= 1u << (i * NH + h);
            tc_fence_after();
            return r;
          };
          auto q_wait = [&](int i) {  // Q tile of group i of the item at q
            const int qi = q.s * NW + i;
            const bool r = wait(&q_full[qi], (ph_q >> qi) & 1);
            ph_q ^= 1u << qi;
            tc_fence_after();
            return r;
          };
          auto take = [&](Item& w) {  // the next item that has keys
            const Item* item;
            while ((item = next(DEVERR_WAIT_MMA)) != nullptr) {
              w = *item;
              done();
              if (w.t0 < w.t1) return true;
            }
            return false;
          };
          Item w, w2;
          if (SHORT) {
            // kv: the K tile of w, then its V tile, then the K tile of w2
            bool have = take(w), loaded = false;
            auto start = [&](const Item& x, int i, const RingPos& k) {  // S of group i of an item
              if (i * 128 >= x.rows) return;
              if (!loaded) ok = wait(&kv_full[k.s], k.ph);
              loaded = true;
              ok = ok && q_wait(i);
              if (ok) issue_s(x, i, q.s * qtiles + i, 0, k.s);
            };
            if (have) {
              for (int i = 0; ok && i < NW; ++i) start(w, i, kv);
              umma_commit(&kv_empty[kv.s]);
              q.advance(p.nq);
            }
            while (ok && have) {
              const bool more = take(w2);
              const RingPos v = kv.next(p.ring), k2 = v.next(p.ring);
              loaded = false;
              ok = v_wait(w, v, 0);
              for (int i = 0; ok && i < NW; ++i) {
                if (i * 128 < w.rows) {
                  if (!(ok = p_wait(i, 0))) break;
                  issue_pv(w, i, 0, 0, v.s, true);
                  umma_commit(&o_full[i]);
                }
                if (more && i > 0) start(w2, i - 1, k2);
              }
              if (!ok) break;
              umma_commit(&kv_empty[v.s]);
              if (more) {
                start(w2, NW - 1, k2);
                umma_commit(&kv_empty[k2.s]);
                q.advance(p.nq);
              }
              kv = k2;
              w = w2;
              have = more;
            }
          } else {
            while (ok && take(w)) {
              const int nw = (w.rows + 127) / 128, qb = q.s * qtiles;
              if (!p.by_keys) {
                if ((ok = wait(&kv_full[kv.s], kv.ph))) {
                  for (int i = 0; ok && i < nw; ++i)
                    if ((ok = q_wait(i))) issue_s(w, i, qb + i, w.t0, kv.s);
                  umma_commit(&kv_empty[kv.s]);
                }
                for (int t = w.t0; ok && t < w.t1; ++t) {  // kv: the K tile of t, then its V tile, then the next K tile
                  const bool more = t + 1 < w.t1;
                  const RingPos v = kv.next(p.ring), k2 = v.next(p.ring);
                  ok = v_wait(w, v, t) && (!more || wait(&kv_full[k2.s], k2.ph));
                  for (int i = 0; ok && i < nw; ++i) {
                    for (int h = 0; ok && h < NH; ++h)
                      if ((ok = p_wait(i, h))) issue_pv(w, i, t, h, v.s, t == w.t0);
                    if (!ok) break;
                    if (more) issue_s(w, i, qb + i, t + 1, k2.s);
                    else umma_commit(&o_full[i]);
                  }
                  if (!ok) break;
                  umma_commit(&kv_empty[v.s]);
                  if (more) umma_commit(&kv_empty[k2.s]);
                  kv = k2;
                }
              } else {
                // group i takes tiles t0 + i, t0 + i + NW, ...: P V of a tile, then S of the group's next one
                ok = q_wait(0);
                RingPos v = kv.next(p.ring);  // V tile of `t`; kv: K tile of `t + NW`
                for (int t = w.t0 - NW; ok && t < w.t1; ++t) {
                  if (t >= w.t0) {
                    const int i = (t - w.t0) % NW;
                    if (!(ok = v_wait(w, v, t))) break;
                    for (int h = 0; ok && h < NH; ++h)
                      if ((ok = p_wait(i, h))) issue_pv(w, i, t, h, v.s, t - w.t0 < NW);
                    if (!ok) break;
                    if (t + NW >= w.t1) umma_commit(&o_full[i]);
                    umma_commit(&kv_empty[v.s]);
                    v = v.next(p.ring).next(p.ring);
                  }
                  if (t + NW < w.t1) {
                    if (!(ok = wait(&kv_full[kv.s], kv.ph))) break;
                    tc_fence_after();
                    issue_s(w, (t + NW - w.t0) % NW, qb, t + NW, kv.s);
                    umma_commit(&kv_empty[kv.s]);
                    kv = kv.next(p.ring).next(p.ring);
                  }
                }
              }
              q.advance(p.nq);
            }
          }
        }
        if (!ok) *abort_flag = 1;
      }
    } else if (svc == 2) {
      RingPos kv;
      bool ok = true;
      for (const Item* item; ok && (item = next_all(DEVERR_WAIT_SOFTMAX));) {
        const Item w = *item;
        __syncwarp();
        if (lane == 0) mbar_arrive_relaxed(&item_empty[ip.s]);
        ip.advance(kItems);
        for (int t = w.t0; ok && t < w.t1; ++t) {
          // Every tile is waited for and given back, cleaned or not: nothing refills it before this warp has seen it, so its
          // phase here is never more than one behind.
          const RingPos k = kv, v = kv.next(p.ring);
          kv = v.next(p.ring);
          ok = __all_sync(0xffffffffu, wait_on(&kv_full[k.s], k.ph, abort_flag, p.err, DEVERR_WAIT_SOFTMAX));
          if (!ok) break;
          if (lane == 0) mbar_arrive_relaxed(&kv_empty[k.s]);
          if (!cleaned(w, t)) {
            ok = __all_sync(0xffffffffu, wait_on(&kv_full[v.s], v.ph, abort_flag, p.err, DEVERR_WAIT_SOFTMAX));
            if (ok && lane == 0) mbar_arrive_relaxed(&kv_empty[v.s]);
            continue;
          }
          const int left = min(w.n - t * KT, KT), reach = (left + 15) / 16 * 16;  // rows that P V reads
          uint32_t off[KT / 32];
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) {
            const int j = c * 32 + lane;
            off[c] = __ballot_sync(0xffffffffu, j < reach && (j >= left || (p.mask && !__ldg(p.mask + (long long)w.b * p.Skv + t * KT + j))));
          }
          ok = __all_sync(0xffffffffu, wait_on(&kv_full[v.s], v.ph, abort_flag, p.err, DEVERR_WAIT_SOFTMAX));
          if (!ok) break;
          uint4* vt = reinterpret_cast<uint4*>(sKV + v.s * C::TILE);
#pragma unroll
          for (int c = 0; c < KT / 32; ++c)
            if (off[c]) {
#pragma unroll
              for (int k = 0; k < 8; ++k)  // four rows at a time: lane / 8 the row, lane % 8 its 16-byte piece
                if ((off[c] >> (k * 4 + lane / 8)) & 1) {
#pragma unroll
                  for (int h = 0; h < D / 64; ++h) vt[h * (C::HALF / 16) + (c * 32 + k * 4) * 8 + lane] = make_uint4(0, 0, 0, 0);
                }
            }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&v_clean[v.s]);
            mbar_arrive_relaxed(&kv_empty[v.s]);
          }
        }
      }
      if (!ok) *abort_flag = 1;
    } else if (svc == 3) {
      if (elect_one()) {
        Items it(p, ends);
        for (Item w = {}; w.rows >= 0; ip.advance(kItems)) {
          const bool more = it.next(w);
          if (!wait_on(&item_empty[ip.s], ip.ph ^ 1, abort_flag, p.err, DEVERR_WAIT_EPI)) {
            *abort_flag = 1;
            break;
          }
          if (!more) w.rows = 0;
          items[ip.s] = w;
          mbar_arrive(&item_full[ip.s]);
          if (!more) break;
        }
      }
    }
  } else {
    if constexpr (!SHORT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFT_REGS));
    // ---------------- softmax warps: one packed row per lane ----------------
    const int i = warp / 4, wq = warp & 3;
    const int lrow = wq * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t tS = tmem + i * C::TCOLS + (static_cast<uint32_t>(wq * 32) << 16), tO = tS + C::TO;
    const int row = p.by_keys ? lrow : i * 128 + lrow;               // row of the item
    const int warp_row = p.by_keys ? wq * 32 : i * 128 + wq * 32;
    const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
    RingPos q;
    unsigned ph_s = 0, ph_o = 0;
    bool ok = true;
    for (const Item* item; ok && (item = next_all(DEVERR_WAIT_SOFTMAX)) != nullptr;) {
      const Item& w = *item;  // read again where it is used: registers are short here
      const int slot = ip.s;
      ip.advance(kItems);
      const bool keys = w.t0 < w.t1;  // the item has a Q tile
      uint8_t* stage = sQ + (q.s * qtiles + (p.by_keys ? 0 : i)) * C::TILE + wq * 4096;
      const RingPos at = q;
      uint64_t* q_done = &q_empty[q.s * NW + (p.by_keys ? 0 : i)];
      if (keys) q.advance(p.nq);
      if (!p.by_keys && i * 128 >= w.rows) {
        __syncwarp();  // every lane has read the item
        if (lane == 0) mbar_arrive_relaxed(&item_empty[slot]);
        continue;
      }
      const bool mine = row < w.rows, warp_on = warp_row < w.rows;
      const int ta = p.by_keys ? w.t0 + i : w.t0, tstep = p.by_keys ? NW : 1;  // this group's key tiles
      const bool any = ta < w.t1;
      float m_run = -INFINITY;
      uint64_t acc[2] = {0, 0};  // sums of the probabilities under m_run
      auto s_wait = [&] {
        const bool r = wait_on(&s_full[i], ph_s, abort_flag, p.err, DEVERR_WAIT_SOFTMAX);
        return __all_sync(0xffffffffu, r);
      };
      auto p_done = [&](int h) {
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[i * NH + h]);
      };
      auto mask = [&](float(&s)[32], int t, int c) {  // -inf for the keys that are masked or past the length
        const int left = w.n - t * KT - c * 32;
        if (__builtin_expect(left >= 32 && !p.mask, 1)) return;
        uint32_t bits = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0;
        if (p.mask)
          bits = __ballot_sync(0xffffffffu, lane < left && __ldg(p.mask + (long long)w.b * p.Skv + t * KT + c * 32 + lane));
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (!((bits >> k) & 1)) s[k] = -INFINITY;
      };
      auto top_of = [&](float (&mx)[4], const float(&s)[32]) {
#pragma unroll
        for (int k = 0; k < 32; k += 2) mx[k / 2 % 4] = max3f(mx[k / 2 % 4], s[k], s[k + 1]);
      };
      // the tile's maximum is at hand: where it passes the one that the exponentials were taken under by more than
      // kRescale, what was made under that one is scaled down (past an item's first tile this is rare)
      auto rescale = [&](const float (&mx)[4], bool first) {
        const float top = fmaxf(max3f(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;  // the scale is positive
        const bool move = top > m_run + kRescale;
        if (__builtin_expect(!__any_sync(0xffffffffu, move), 1)) return;
        const float m_new = move ? top : m_run, alpha = move ? ex2_approx(m_run - m_new) : 1.0f;
        const uint64_t al2 = f2_pack(alpha, alpha);
        m_run = m_new;
        acc[0] = mul2(acc[0], al2);
        acc[1] = mul2(acc[1], al2);
        if (first) return;
        // this tile's scores follow the last P V on the tensor pipe: O is complete
#pragma unroll 1
        for (int j = 0; j < D / 16; ++j) {
          uint32_t r[16];
          tmem_ld16(tO + j * 16, r);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const uint64_t x = mul2(f2_pack(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), al2);
            r[k] = (uint32_t)x;
            r[k + 1] = (uint32_t)(x >> 32);
          }
          tmem_st16(tO + j * 16, r);
        }
      };
      auto exps = [&](float(&s)[32], uint32_t tP) {  // probabilities, in place (32 scores -> 16 words) and into TMEM
        const float m_sub = m_run == -INFINITY ? 0.f : m_run;  // no valid key yet: every p is 2^-inf = 0
        const uint64_t nm2 = f2_pack(-m_sub, -m_sub);
        uint32_t* w32 = reinterpret_cast<uint32_t*>(s);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const uint64_t x = fma2(f2_pack(s[k], s[k + 1]), sc2, nm2);
          const float a = ex2_approx(lo_f(x)), b = ex2_approx(hi_f(x));
          acc[k / 2 % 2] = add2(acc[k / 2 % 2], f2_pack(a, b));
          w32[k / 2] = pack2<BF16>(a, b);
        }
        tmem_st16(tP, w32);
      };
      auto load = [&](float(&s)[32], int c) { tmem_ld32(tS + c * 32, reinterpret_cast<uint32_t(&)[32]>(s)); };
#pragma unroll 1
      for (int t = ta; t < w.t1; t += tstep) {
        ok = s_wait();
        if (!ok) break;
        tc_fence_after();
        if constexpr (SHORT) {
          // Two passes over the scores in TMEM, 32 at a time: the maximum, then the exponentials.  Loops, not unrolled: with
          // three groups the code of a tile has to stay in the instruction caches that all roles share.
          if (warp_on) {
            const int nc = (w.n + 31) / 32;
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (int c = 0; c < nc; ++c) {
              float s[32];
              load(s, c);
              wait_ld(s);
              mask(s, t, c);
              top_of(mx, s);
            }
            rescale(mx, true);
#pragma unroll 1
            for (int c = 0; c < nc; ++c) {
              float s[32];
              load(s, c);
              wait_ld(s);
              mask(s, t, c);
              exps(s, tS + c * 16);  // over the scores of chunk c / 2
            }
          }
          p_done(0);
        } else if (!warp_on) {
          p_done(0);
          p_done(1);
        } else {
          // The tile's scores are read once and stay in registers: every trip to TMEM costs 150 cycles, a second pass
          // over the scores made this 4300 cycles a tile and group pair instead of 3600.  P of the tile's first half is
          // handed over while the exponentials of the second run.
          float s0[32], s1[32], s2[32], s3[32];
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          load(s0, 0);
          load(s1, 1);
          load(s2, 2);
          load(s3, 3);
          wait_ld(s0);
          wait_ld(s1);
          wait_ld(s2);
          wait_ld(s3);
          if (__builtin_expect(p.mask || w.n - t * KT < KT, 0)) {
            mask(s0, t, 0);
            mask(s1, t, 1);
            mask(s2, t, 2);
            mask(s3, t, 3);
          }
          top_of(mx, s0);
          top_of(mx, s1);
          top_of(mx, s2);
          top_of(mx, s3);
          rescale(mx, t == ta);
          exps(s0, tS);
          exps(s1, tS + 16);
          p_done(0);
          exps(s2, tS + 32);
          exps(s3, tS + 48);
          p_done(1);
        }
        ph_s ^= 1;
      }
      const uint64_t sum = add2(acc[0], acc[1]);
      const float l_run = lo_f(sum) + hi_f(sum);
      if (ok && any) {
        ok = wait_on(&o_full[i], ph_o, abort_flag, p.err, DEVERR_WAIT_SOFTMAX);
        ok = __all_sync(0xffffffffu, ok);
        ph_o ^= 1;
        tc_fence_after();
      }
      if (!ok) break;
      bool staged = false;
      if (warp_on) {
        const long long pr = ((long long)w.slot * NW + i) * 128 + lrow;  // by keys: the row's partial
        const int tr = w.row0 + row;                                     // packed row of the group
        const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
        const uint64_t inv2 = f2_pack(inv, inv);
        staged = !p.by_keys && any && warp_row + 32 <= w.rows;
        uint16_t* o = static_cast<uint16_t*>(p.O) + w.b * p.osb + (tr >> p.gps) * p.oss +
                      ((w.hg << p.gps) + (tr & (p.GP - 1))) * p.osh;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          if (any) {  // warp-uniform
            tmem_ld32(tO + c * 32, r);
            tmem_wait_ld();
          }
          if (SHORT && c == D / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (any && lane == 0) mbar_arrive_relaxed(&o_read[i]);
          }
          if (p.by_keys) {
            if (mine && any) {
              float4* d = reinterpret_cast<float4*>(p.part + pr * D + c * 32);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                d[k] = make_float4(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1]),
                                   __uint_as_float(r[4 * k + 2]), __uint_as_float(r[4 * k + 3]));
            }
            continue;
          }
          uint32_t h[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {  // no valid key: zeros, whatever O holds
            const uint64_t x = mul2(f2_pack(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1])), inv2);
            h[k] = l_run == 0.f ? 0u : pack2<BF16>(lo_f(x), hi_f(x));
          }
          if (staged) {  // 128-byte swizzled rows, 64 columns to a half tile
            uint4* d = reinterpret_cast<uint4*>(stage + c / 2 * C::HALF + lane * 128);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              d[(c % 2 * 4 + k) ^ (lane & 7)] = make_uint4(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
          } else if (mine) {
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
        if (p.by_keys && mine)
          reinterpret_cast<float2*>(p.part + (long long)p.slots * NW * 128 * D)[pr] = make_float2(m_run, l_run);
        if (staged) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int tr0 = w.row0 + warp_row;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_store_5d(&p.tmO, stage + c * C::HALF, c * 64, tr0 & (p.GP - 1), tr0 >> p.gps, w.hg, w.b);
            bulk_commit();
            bulk_wait_read0();
          }
        }
      } else if (SHORT && any && lane == 0) {
        mbar_arrive_relaxed(&o_read[i]);
      }
      // By keys all groups release the one Q tile.  A group without a key tile waits until it has landed: running ahead, it
      // would release the buffer's next tile in another group's place.
      if (p.by_keys && keys && !any) {
        ok = __all_sync(0xffffffffu, wait_on(&q_full[at.s * NW], at.ph, abort_flag, p.err, DEVERR_WAIT_SOFTMAX));
        if (!ok) break;
      }
      tc_fence_before();  // O is read before the next item's first P V, which waits for this warp's p_full
      __syncwarp();
      if (lane == 0) {
        if (keys) mbar_arrive_relaxed(q_done);
        mbar_arrive_relaxed(&item_empty[slot]);
      }
    }
    if (!ok) *abort_flag = 1;
    if (lane == 0) bulk_wait0();
  }
  tc_fence_before();
  __syncthreads();
  if (svc == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the keys: one warp per packed row.
template <bool BF16, int D>
__global__ void __launch_bounds__(128) xattn_join_kernel(const __grid_constant__ XattnParams p) {
  constexpr int NW = XCfg<D, false>::NW;
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const int pair = (int)(blockIdx.y);  // (b, hg, row block)
  const int b = pair / p.RT / p.HG, hg = pair / p.RT % p.HG, rt = pair % p.RT;
  const int lrow = blockIdx.x * 4 + threadIdx.x / 32, t = rt * 128 + lrow;
  const int q = p.q_len ? min(max(__ldg(p.q_len + b), 0), p.Sq) : p.Sq;
  if (t >= q << p.gps) return;
  // this block's place in the key tiles laid end to end, and the CTAs that share it
  int before = 0, total = 0, nt = 0;
  for (int x = lane; x < p.B; x += 32) {
    const int n = ((p.kv_len ? min(max(__ldg(p.kv_len + x), 0), p.Skv) : p.Skv) + KT - 1) / KT;
    total += n;
    if (x < b) before += n;
    if (x == b) nt = n;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
    nt += __shfl_xor_sync(0xffffffffu, nt, o);
  }
  const long long all = (long long)total * p.HG * p.RT;
  const long long g0 = (long long)before * p.HG * p.RT + (long long)(pair - b * p.HG * p.RT) * nt, g1 = g0 + nt;
  float m = -INFINITY, l = 0.f;
  constexpr int W = D / 32;
  float acc[W] = {};
  if (nt) {
    // CTA c has tiles [all c / grid, all (c + 1) / grid): the first and last that meet [g0, g1)
    int c0, c1;
    if (all * p.grid < 1ll << 31) {  // 32-bit divisions take a tenth of the time
      c0 = ((int)(g0 + 1) * p.grid - 1) / (int)all;
      c1 = ((int)g1 * p.grid - 1) / (int)all;
    } else {
      c0 = (int)(((g0 + 1) * p.grid - 1) / all);
      c1 = (int)((g1 * p.grid - 1) / all);
    }
    const float2* ml = reinterpret_cast<const float2*>(p.part + (long long)p.slots * NW * 128 * D);
    const int n = (c1 - c0 + 1) * NW;
    const long long base = ((long long)(c0 + pair) * NW) * 128 + lrow;
    auto part_of = [&](int s) {  // (max, sum) of part s; sum 0: nothing valid there, its O may not even be written
      if (s >= n) return make_float2(-INFINITY, 0.f);
      const long long c = c0 + s / NW;  // fewer tiles than CTAs: some have none
      if (all < p.grid && all * c / p.grid == all * (c + 1) / p.grid) return make_float2(-INFINITY, 0.f);
      return ml[base + s * 128];
    };
    const float2 first = part_of(lane);
    if (first.y != 0.f) m = first.x;
    for (int s = lane + 32; s < n; s += 32) {
      const float2 v = part_of(s);
      if (v.y != 0.f) m = fmaxf(m, v.x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int s0 = 0; s0 < n; s0 += 32) {
      const float2 v = s0 ? part_of(s0 + lane) : first;
      const float mine = v.y != 0.f ? ex2_approx(v.x - m) : 0.f;  // NaN passes
      if (v.y != 0.f) l = fmaf(v.y, mine, l);
      const unsigned with = __ballot_sync(0xffffffffu, v.y != 0.f);
      for (int j0 = 0; j0 < min(n - s0, 32); j0 += 8) {  // eight parts' loads in flight
        uint32_t o[8][W];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t* src = reinterpret_cast<const uint32_t*>(p.part + (base + (s0 + j0 + j) * 128) * D + lane * W);
#pragma unroll
          for (int k = 0; k < W; ++k) o[j][k] = (with >> (j0 + j)) & 1 ? src[k] : 0u;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f = __shfl_sync(0xffffffffu, mine, j0 + j);
#pragma unroll
          for (int k = 0; k < W; ++k) acc[k] = fmaf(__uint_as_float(o[j][k]), f, acc[k]);
        }
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t* o = static_cast<uint16_t*>(p.O) + b * p.osb + (t >> p.gps) * p.oss +
                ((hg << p.gps) + (t & (p.GP - 1))) * p.osh + lane * W;
#pragma unroll
  for (int k = 0; k < W; k += 2) reinterpret_cast<uint32_t*>(o)[k / 2] = pack2<BF16>(acc[k] * inv, acc[k + 1] * inv);
}

struct XPlan {
  int GP, HG, RT, tpi, by_keys, grid, slots;
};
XPlan xattn_plan(const Ctx* c, int B, int H, int Hkv, int Sq, int Skv, int D) {
  XPlan x = {};
  const int G = H / Hkv, NW = D == 64 && Skv <= KT ? 3 : 2;
  x.GP = G & -G;  // packed heads: the power of two in the group (tiles of 128 rows hold whole tokens)
  if (x.GP > 128) x.GP = 128;
  x.HG = H / x.GP;
  const long long rows = (long long)Sq * x.GP, tiles = (rows + 127) / 128, nt = ((long long)Skv + KT - 1) / KT;
  // By rows: as many row tiles per item as fill the SMs in the fewest rounds (an item costs a share of its
  // latency however many tiles it has).
  double best = 1e30;
  for (int n = 1; n <= NW; ++n) {
    const long long items = (long long)B * x.HG * ((tiles + n - 1) / n);
    const double cost = (double)((items + c->num_sms - 1) / c->num_sms) * (2.0 + n);
    if (cost <= best) {
      best = cost;
      x.tpi = n;
    }
  }
  // By keys where that is estimated to be sooner, in microseconds as measured: 5 to start and end and 1.5 for a key tile of
  // one group, 1.9 for one of each of two that take turns; 6 more and the parts' bytes, out and in, to join them.  (112
  // blocks of 2 rows, 4185 keys, head dim 64: 28 by keys, 56 by rows; 72 blocks of 77 rows, 513 keys: 16 and 13.)
  const long long blocks = (long long)B * x.HG * tiles;
  if (blocks <= c->num_sms && nt >= 4 && B <= kMaxByKeys && nt * blocks < (1ll << 30)) {
    const int grid = (int)std::min<long long>(c->num_sms, blocks * nt / 2);
    const double parts = (double)(grid + blocks) * 2 * std::min<long long>(rows, 128) * (D + 2) * 4;
    const double by_rows = 5 + nt * (x.tpi == 1 ? 1.5 : 1.9) * (D == 128 ? 1.15 : 1.0);
    const double by_keys = 11 + (double)((blocks * nt + grid - 1) / grid) * 0.95 + 2 * parts / 6.5e6;
    if (by_keys < by_rows) {
      x.by_keys = 1;
      x.tpi = 1;
      x.RT = (int)tiles;
      x.grid = grid;
      x.slots = grid + (int)blocks;
      return x;
    }
  }
  x.RT = (int)((tiles + x.tpi - 1) / x.tpi);
  return x;
}

template <bool BF16, int D, bool SHORT>
int launch_xattn(Ctx* c, XattnParams& p) {
  using C = XCfg<D, SHORT>;
  auto kern = xattn_kernel<BF16, D, SHORT>;
  static unsigned attr_done = 0;
  if (!(attr_done & (1u << (c->device & 31)))) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::TOTAL) != cudaSuccess)
      return cudaGetLastError(), set_error(c, DI_ECUDA, "cross_attention: shared memory attribute");
    // the softmax warps' registers come out of the launch's: too few would leave them waiting for more
    cudaFuncAttributes a = {};
    if (!SHORT && (cudaFuncGetAttributes(&a, kern) != cudaSuccess ||
                   a.numRegs * C::THREADS < 32 * (C::SW * C::SOFT_REGS + 4 * C::SERVICE_REGS)))
      return cudaGetLastError(), set_error(c, DI_ECUDA, "cross_attention: built with too few registers");
    attr_done |= 1u << (c->device & 31);
  }
  const int qtiles = p.by_keys ? 1 : p.tpi;
  // Q of the next item is fetched under this one where a ring of four tiles remains
  p.nq = std::max(1, std::min<int>(SHORT ? kQBufs : 2, (int)(C::DATA / C::TILE - 4) / qtiles));
  p.ring = (int)std::min<uint32_t>(C::MAXRING, (C::DATA - p.nq * qtiles * C::TILE) / C::TILE);
  const unsigned grid = p.by_keys ? p.grid : std::min<unsigned>(p.items, c->num_sms);
  if (!p.by_keys) {
    p.d_rt = (int)(grid % p.RT);
    p.d_hg = (int)(grid / p.RT % p.HG);
    p.d_b = (int)(grid / p.RT / p.HG);
  }
  launch_k(kern, dim3(grid), C::THREADS, C::TOTAL, c->stream, p);
  if (p.by_keys) {
    const int rc = check_launch(c, "cross_attention");
    if (rc != DI_OK) return rc;
    const int rows = (int)std::min<long long>(128, (long long)p.Sq << p.gps);
    launch_k(xattn_join_kernel<BF16, D>, dim3((rows + 3) / 4, p.B * p.HG * p.RT), 128, 0, c->stream, p);
  }
  return check_launch(c, "cross_attention");
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" size_t di_cross_attention_workspace(di_ctx_t h, const long long cfg[18]) {
  if (!h || !cfg) return 0;
  for (int i = 0; i < 6; ++i)
    if (cfg[i] <= 0 || cfg[i] > (1ll << 30)) return 0;
  const int B = (int)cfg[0], H = (int)cfg[1], Hkv = (int)cfg[2], D = (int)cfg[5];
  if (H % Hkv || (D != 64 && D != 128)) return 0;
  const XPlan x = xattn_plan(ctx_of(h), B, H, Hkv, (int)cfg[3], (int)cfg[4], D);
  return (size_t)x.slots * 2 * 128 * (D + 2) * 4;
}

extern "C" int di_cross_attention(di_ctx_t h, int dtype, const long long cfg[18], float scale, const void* Q, const void* K,
                                  const void* V, void* O, const int* q_len, const int* kv_len,
                                  const unsigned char* key_mask, void* ws, size_t ws_bytes) {
  Ctx* c = ctx_of(h);
  if (!c || (dtype != DI_F16 && dtype != DI_BF16)) return DI_EINVAL;
  DeviceGuard guard(c->device);
  if (!cfg || !Q || !K || !V || !O) return set_error(c, DI_EINVAL, "cross_attention: bad shape or missing tensor");
  for (int i = 0; i < 6; ++i)
    if (cfg[i] <= 0 || cfg[i] > (1ll << 30)) return set_error(c, DI_EINVAL, "cross_attention: bad shape or missing tensor");
  const int B = (int)cfg[0], H = (int)cfg[1], Hkv = (int)cfg[2], Sq = (int)cfg[3], Skv = (int)cfg[4], D = (int)cfg[5];
  const long long *q_strides = cfg + 6, *k_strides = cfg + 9, *v_strides = cfg + 12, *o_strides = cfg + 15;
  if (H % Hkv) return set_error(c, DI_EINVAL, "cross_attention: H must be a multiple of Hkv");
  if (D != 64 && D != 128) return set_error(c, DI_EUNSUPPORTED, "cross_attention: head dim must be 64 or 128");
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(O))
    return set_error(c, DI_EINVAL, "cross_attention: pointers must be 16-byte aligned");
  const XPlan x = xattn_plan(c, B, H, Hkv, Sq, Skv, D);
  if ((long long)Sq * x.GP > (1 << 30) || (long long)B * x.HG * x.RT > 0x7fffffffll)
    return set_error(c, DI_EUNSUPPORTED, "cross_attention: too many tokens");
  // strides of axes of length one mean nothing: they are replaced by 8 elements (a valid tensor-map stride)
  long long qs[3], ks[3], vs[3], os[3];
  bool same = true;  // Q and O in one layout
  for (int i = 0; i < 3; ++i) {
    const int nq = i == 0 ? B : i == 1 ? Sq : H, nk = i == 0 ? B : i == 1 ? Skv : Hkv;
    qs[i] = nq > 1 ? q_strides[i] : 8;
    ks[i] = nk > 1 ? k_strides[i] : 8;
    vs[i] = nk > 1 ? v_strides[i] : 8;
    os[i] = nq > 1 ? o_strides[i] : 16;
    same = same && (nq == 1 || qs[i] == os[i]);
    if (qs[i] < 0 || ks[i] < 0 || vs[i] < 0 || (qs[i] | ks[i] | vs[i] | os[i]) % 8 || os[i] < 0)
      return set_error(c, DI_EINVAL, "cross_attention: strides must be multiples of 8 elements and not negative");
    if (os[i] == 0) return set_error(c, DI_EINVAL, "cross_attention: the output's rows must not share memory");
  }
  if (qs[1] == 0 || ks[1] == 0 || vs[1] == 0 || (qs[2] == 0 && x.GP > 1))
    return set_error(c, DI_EINVAL, "cross_attention: tokens and grouped query heads cannot be expanded");
  if (!(scale > 0.f) || !(scale < INFINITY)) return set_error(c, DI_EINVAL, "cross_attention: scale must be positive and finite");
  const size_t need = di_cross_attention_workspace(h, cfg);
  if (need && (!ws || ws_bytes < need || !aligned16(ws)))
    return set_error(c, DI_EINVAL, "cross_attention: workspace missing, too small or not 16-byte aligned");
  // an item's queries are read before its rows are written, but its keys and values serve other items too
  if (O == K || O == V || (O == Q && !same))
    return set_error(c, DI_EINVAL, "cross_attention: the output shares memory with k, v, or queries in another layout");
  XattnParams p;
  memset(&p, 0, sizeof p);
  const CUtensorMapDataType dt = dtype == DI_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  std::string err;
  // an expanded axis (stride 0) becomes an axis of length one whose coordinate stays 0
  auto len = [](long long stride, int n) { return (uint64_t)(stride ? n : 1); };
  auto str = [](long long stride) { return (uint64_t)(stride ? stride : 8) * 2; };
  const uint64_t qd[5] = {(uint64_t)D, (uint64_t)x.GP, (uint64_t)Sq, len(qs[2], x.HG), len(qs[0], B)};
  const uint64_t qst[4] = {str(qs[2]), str(qs[1]), str(qs[2] * x.GP), str(qs[0])};
  const uint32_t qbox[5] = {64, (uint32_t)x.GP, (uint32_t)(128 / x.GP), 1, 1};
  const bool is_short = D == 64 && Skv <= KT;
  const uint32_t kbox[4] = {64, KT, 1, 1};
  const uint64_t kd[4] = {(uint64_t)D, (uint64_t)Skv, len(ks[2], Hkv), len(ks[0], B)};
  const uint64_t vd[4] = {(uint64_t)D, (uint64_t)Skv, len(vs[2], Hkv), len(vs[0], B)};
  const uint64_t kst[3] = {str(ks[1]), str(ks[2]), str(ks[0])}, vst[3] = {str(vs[1]), str(vs[2]), str(vs[0])};
  const uint64_t od[5] = {(uint64_t)D, (uint64_t)x.GP, (uint64_t)Sq, (uint64_t)x.HG, (uint64_t)B};
  const uint64_t ost[4] = {str(os[2]), str(os[1]), str(os[2] * x.GP), str(os[0])};
  const uint32_t gbox = std::min(x.GP, 32);
  const uint32_t obox[5] = {64, gbox, 32 / gbox, 1, 1};  // a warp's 32 rows
  if (!make_tmap(&p.tmQ, dt, 5, Q, qd, qst, qbox, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmK, dt, 4, K, kd, kst, kbox, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmV, dt, 4, V, vd, vst, kbox, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmO, dt, 5, O, od, ost, obox, CU_TENSOR_MAP_SWIZZLE_128B, &err))
    return set_error(c, DI_EINVAL, "cross_attention: " + err);
  p.qh_mul = qs[2] != 0; p.qb_mul = qs[0] != 0;
  p.kh_mul = ks[2] != 0; p.kb_mul = ks[0] != 0;
  p.vh_mul = vs[2] != 0; p.vb_mul = vs[0] != 0;
  p.O = O;
  p.osb = os[0]; p.oss = os[1]; p.osh = os[2];
  p.wide = (reinterpret_cast<uintptr_t>(O) & 31) == 0 && (os[0] | os[1] | os[2]) % 16 == 0;
  while ((1 << p.gps) < x.GP) ++p.gps;
  p.B = B; p.HG = x.HG; p.GP = x.GP; p.G = H / Hkv; p.Sq = Sq; p.Skv = Skv; p.RT = x.RT; p.tpi = x.tpi;
  p.by_keys = x.by_keys; p.grid = x.grid; p.slots = x.slots;
  p.items = (unsigned)B * x.HG * x.RT;
  p.q_len = q_len; p.kv_len = kv_len; p.mask = key_mask;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.part = static_cast<float*>(ws);
  p.err = c->d_err;
  if (dtype == DI_F16) {
    if (D == 128) return launch_xattn<false, 128, false>(c, p);
    return is_short ? launch_xattn<false, 64, true>(c, p) : launch_xattn<false, 64, false>(c, p);
  }
  if (D == 128) return launch_xattn<true, 128, false>(c, p);
  return is_short ? launch_xattn<true, 64, true>(c, p) : launch_xattn<true, 64, false>(c, p);
}
