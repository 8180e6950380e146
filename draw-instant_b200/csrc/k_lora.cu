// k_lora.cu — a linear layer with a low-rank adapter per row beside the shared weight (sm_100a).
//
//   Y[m] = act(X[m] W^T + bias + scale[a] (X[m] A[a]^T) B[a]^T) + R[m],   a = row_adapter[m]
//
// A negative index takes no adapter; an index past the last adapter takes none either and sets
// DEVERR_BOUNDS in the device error word.
//
// Two launches.  The first computes T = scale[a] X A[a]^T, a row's own `rank` values; the second is the product with
// W and adds T B[a]^T.  The first kernel lets the second start as soon as its own wait for earlier kernels is over, so the
// second reads X and W at once and waits only before it reads T.
//
// Tiles (M > kSkinnyRows): T is kept as two 16-bit parts, hi + lo (2^-17 relative for bf16), and is simply more of K:
// after the K blocks of X and W come, for every adapter that the tile's rows name, a block of [T_hi | T_lo] against that
// adapter's B, with the T rows of other adapters zeroed in shared memory.  A tile may so mix adapters at the price of a
// block each.  (tcgen05.mma's own mask of output lanes would spare the zeroing, but a masked MMA took some 1000 cycles, whatever
// its width, against 80 to 128 for a plain one.)  Zero times an infinity or NaN in another adapter's B is NaN: outputs
// that are not finite in a tile of several adapters are computed again from their own row's terms alone (1001 x 1024 x 4096,
// rank 64, with every row NaN: 180 us instead of 29).  In a tile of one adapter they stand: an infinity in its B may come
// out as NaN there, T's two parts having signs of their own.
// One persistent CTA per SM, or CTA pair (cta_group::2: 256 rows, each CTA loads half of B):
//   warp 0       TMA loads through one ring of stages
//   warp 1       MMA issue (the pair's first CTA)
//   warp 2       the tile's distinct adapters and the rows of each
//   warp 3       zeroes other adapters' rows of a T block
//   warps 4-15   epilogue: bias, activation, residual (fetched by TMA a chunk ahead), stores from registers
// The accumulator is double-buffered, so a tile's epilogue runs under the next one's main loop.
//
// Few rows (M <= kSkinnyRows): T in 32 bits (in shared memory, with no first launch, where that is less work); the second
// launch streams W into mma.sync fragments (16 weight rows by 8 rows of X) and adds the rows' own B products with plain
// FMAs: every byte of W, A and B comes from memory once, whoever owns it.
//
// Bound and measured (graph replays).  Tiles: 65536 x 320 x 320, rank 32, residual, fp16: 40.6 us, 3.1 TB/s (the shared
// product alone 33); 16384 x 640 x 1920, rank 16: 49 us, 845 TFLOP/s; 1001 x 1024 x 4096, rank 64, six adapters, gelu:
// 24.2 us.  Neither memory nor the tensor pipe is full: a tile's k blocks, T blocks, zeroing and epilogue hand over to one
// another some ten times, 150 to 300 ns each (without the epilogue the first takes 29.6 us, with a quarter of the MMAs
// 40.8).  T as a second kernel's work costs 2.5 to 9 us.
// Few rows: 8 x 1280 x 1280, rank 16: 4.6 us; 64 x 1024 x 4096, rank 32, 64 adapters: 12.0 us, 2.3 TB/s; bound by the
// latency of one pass (two launches, one batch of loads each) and, towards 128 rows, by X from L2 for every 32 columns.
#include <algorithm>
#include <cstring>

#include "di_common.cuh"

namespace di {

struct LoraParams {
  CUtensorMap tmX, tmW, tmA, tmT, tmB, tmR;
  const void *X, *W, *A, *B, *R;
  void* Y;
  long long ldx, ldr, ldy;
  int M, N, K, r, L;
  const float *scale, *bias;
  const int* rows;
  int act;
  int* err;
  // tiles
  int BN, stages, mt, nt;
  int wide;             // rows of Y take 32-byte stores
  uint32_t stage_bytes;
  int tslots, tstages;  // first kernel: adapters per pass
  uint32_t tstage_bytes;
  uint16_t* T16;  // [M][t_ld]: 64-column groups, hi and lo parts of 32 ranks (r <= 32) or of 64 in two groups
  int t_ld;
  // few rows
  float* T;       // [M][r]
};

namespace {

constexpr int kSkinnyRows = 128;
constexpr int kEpi = 12;           // epilogue warps: three share a quarter of the rows, 32-column chunks in turn
constexpr int kEpiPer = kEpi / 4;
constexpr int kLThreads = 128 + 32 * kEpi, kTThreads = 256;
constexpr int kMaxStages = 12;
constexpr int kSlots = 32;        // adapters per list entry
constexpr int kLists = 3;
constexpr int kSlabs = 2;         // residual slabs per epilogue warp
constexpr uint32_t kSlab = 2048;  // 32 x 32 16-bit values

struct SlotList {
  int n, more;               // adapters here; more of the tile's adapters follow in the next entry
  int ids[kSlots];
  uint32_t others[kSlots][8];  // rows of the tile (accumulator lanes) that do not name the adapter
};
constexpr uint32_t kListBytes = (kLists * sizeof(SlotList) + 15) / 16 * 16;
constexpr uint32_t kBarBytes = 8 * (4 * kMaxStages + 2 * kLists + 4 + kEpi * kSlabs) + 16;
constexpr uint32_t kTFixedSmem = 1024 + kListBytes + 8 * (2 * kMaxStages + 2 * kLists + 4) + 32;
constexpr uint32_t kFixedSmem = 1024 + kEpi * 256 + kListBytes + (kBarBytes + 15) / 16 * 16;

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
template <bool PAIR>
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
  if (PAIR) {
    tma_load_2d_pair(dst, m, bar, c0, c1);
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  }
}
template <bool PAIR>
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
        "%5}], [%2];" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
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
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  return BF16 ? __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)) : __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
  return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ float lo_f(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_f(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
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
__device__ __forceinline__ float ex2_approx(float x) {  // 2^x; -inf -> +0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float silu_fast(float v) { return __fdividef(v, 1.0f + __expf(-v)); }
// erf GELU of two values: v Phi(v) = max(v, 0) - |v| Phi(-|v|), and log2 Phi(-a) is so smooth that a polynomial of degree
// 6 (minimax fit on [0, 5.5] for the error of a Phi(-a)) gives the result within 1e-7: one exponential and no
// division per value, half the special-function work of a rational approximation.  Past 5.5 the exponent falls
// on at a slope of 8 (the product is below 1e-7 there and stays so).
__device__ __forceinline__ uint64_t gelu2(uint64_t v) {
  const float v0 = lo_f(v), v1 = hi_f(v), a0 = fabsf(v0), a1 = fabsf(v1), c0 = fminf(a0, 5.5f), c1 = fminf(a1, 5.5f);
  const uint64_t c = f2_pack(c0, c1);
  auto k = [](float x) { return f2_pack(x, x); };
  uint64_t q = fma2(k(3.4440247e-05f), c, k(-0.000778908085f));
  q = fma2(q, c, k(0.00810599886f));
  q = fma2(q, c, k(-0.0534412861f));
  q = fma2(q, c, k(-0.458756894f));
  q = fma2(q, c, k(-1.15120339f));
  q = fma2(q, c, k(-0.999993265f));
  q = fma2(f2_pack(a0 - c0, a1 - c1), k(-8.0f), q);
  return f2_pack(fmaf(-c0, ex2_approx(lo_f(q)), fmaxf(v0, 0.f)), fmaf(-c1, ex2_approx(hi_f(q)), fmaxf(v1, 0.f)));
}
__device__ __forceinline__ float act_of(float v, int act) {
  return act == 1 ? silu_fast(v) : act == 2 ? lo_f(gelu2(f2_pack(v, 0.f))) : v;
}
template <bool BF16>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Buffer index and phase of a ring.
struct Ring {
  int s = 0, ph = 0;
  __device__ __forceinline__ void advance(int n) {
    if (++s == n) { s = 0; ph ^= 1; }
  }
  __device__ __forceinline__ void back(int n) {
    if (--s < 0) { s = n - 1; ph ^= 1; }
  }
};

// K-major operand descriptor of a 128-byte-swizzled tile at shared address `a`; + 2 steps 16 values along K.
__device__ __forceinline__ uint64_t kdesc(uint32_t a) { return sdesc_sw128(0, 16, 1024) | (a >> 4); }

// Bounded wait that also ends when another role has given up; the flag is read only when the phase is not there yet.
template <bool CLUSTER>
__device__ __forceinline__ bool wait_on(uint64_t* bar, int ph, volatile int* abort_flag, int* err, int code) {
  const uint32_t a = smem_u32(bar);
  if (CLUSTER ? mbar_try_wait_cluster(a, ph) : mbar_try_wait(a, ph)) return true;
  return !*abort_flag && mbar_wait<CLUSTER>(bar, ph, err, code);
}

// One warp lists a tile's adapters (rows m0 .. m0 + 32 RL - 1), at most `most` to an entry, with the rows that do not
// name each.  Every tile has one entry at least.
template <int RL>
__device__ __forceinline__ void rows_of(const LoraParams& p, int m0, int lane, int (&a)[RL]) {
#pragma unroll
  for (int i = 0; i < RL; ++i) {
    const int m = m0 + i * 32 + lane;
    a[i] = m < p.M && m0 >= 0 ? __ldg(p.rows + m) : -1;
  }
}
// `next` holds the rows' adapters on entry, and those of the tile at next_m0 (-1: none) on return: a load under the
// traffic of the streams takes microseconds, so it is made a tile ahead.
template <int RL>
__device__ __forceinline__ bool list_adapters(const LoraParams& p, int next_m0, int (&next)[RL], int most, SlotList* lists,
                                              uint64_t* list_full, uint64_t* list_empty, Ring& li,
                                              volatile int* abort_flag, int lane) {
  int a[RL];
#pragma unroll
  for (int i = 0; i < RL; ++i) {
    a[i] = next[i];
    if (a[i] >= p.L) {
      atomicOr(p.err, DEVERR_BOUNDS);
      a[i] = -1;
    }
  }
  rows_of<RL>(p, next_m0, lane, next);
  int n = 0;
  auto open_entry = [&] {
    n = 0;
    return __all_sync(0xffffffffu, wait_on<false>(&list_empty[li.s], li.ph ^ 1, abort_flag, p.err, DEVERR_WAIT_EPI)) != 0;
  };
  auto close_entry = [&](int more) {
    if (lane == 0) {
      lists[li.s].n = n;
      lists[li.s].more = more;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&list_full[li.s]);
    li.advance(kLists);
  };
  if (!open_entry()) return false;
#pragma unroll
  for (int i = 0; i < RL; ++i) {
    unsigned open;
    while ((open = __ballot_sync(0xffffffffu, a[i] >= 0)) != 0) {
      if (n == most) {
        close_entry(1);
        if (!open_entry()) return false;
      }
      const int id = __shfl_sync(0xffffffffu, a[i], __ffs(open) - 1);
#pragma unroll
      for (int k = 0; k < RL; ++k) {
        const unsigned o = __ballot_sync(0xffffffffu, a[k] != id);
        if (a[k] == id) a[k] = -1;
        if (lane == 0) lists[li.s].others[n][k] = o;
      }
      if (lane == 0) lists[li.s].ids[n] = id;
      ++n;
    }
  }
  close_entry(0);
  return true;
}

// ---- tiles: T = scale X A^T in two 16-bit parts ----

// One pass over X per entry of the tile's list (all of its adapters as a rule): the A rows of up to `tslots` adapters are
// the B operand, side by side, and every row keeps its own adapter's columns.  Bound: the bytes of X, which five
// stages per SM stream (more only lengthen the queue that every load waits in).
//   warp 0 TMA loads, warp 1 MMA issue, warp 2 lists, warps 4-7 T out of TMEM, one row per thread
template <bool BF16>
__global__ void __launch_bounds__(kTThreads, 1) lora_t_kernel(const __grid_constant__ LoraParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sStage = smem;  // [tstages]: 128 rows of X, then the adapters' rows, 128 bytes each
  SlotList* lists = reinterpret_cast<SlotList*>(smem + p.tstages * p.tstage_bytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(lists) + kListBytes);  // [kMaxStages]
  uint64_t* empty = full + kMaxStages;         // [kMaxStages]
  uint64_t* list_full = empty + kMaxStages;    // [kLists]
  uint64_t* list_empty = list_full + kLists;   // [kLists]
  uint64_t* d_full = list_empty + kLists;      // [2]
  uint64_t* d_empty = d_full + 2;              // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.tstages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < kLists; ++i) { mbar_init(&list_full[i], 1); mbar_init(&list_empty[i], 6); }
    for (int i = 0; i < 2; ++i) { mbar_init(&d_full[i], 1); mbar_init(&d_empty[i], 4); }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // accumulator ab at column 256 ab
  pdl_begin();
  const int tiles = (p.M + 127) / 128, nk = p.K / 64, rp = (p.r + 15) / 16 * 16;

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tmX);
      tma_prefetch_desc(&p.tmA);
      Ring st, li;
      bool ok = true;
      unsigned issued = 0;
      for (int u = blockIdx.x; ok && u < tiles; u += gridDim.x)
        for (bool more = true; ok && more;) {
          if (!(ok = wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_TMA))) break;
          const SlotList& l = lists[li.s];
          more = l.more;
          for (int kb = 0; l.n && kb < nk; ++kb) {
            if (!(ok = wait_on<false>(&empty[st.s], st.ph ^ 1, abort_flag, p.err, DEVERR_WAIT_TMA))) break;
            uint8_t* d = sStage + st.s * p.tstage_bytes;
            mbar_arrive_expect_tx(&full[st.s], 16384u + (uint32_t)(l.n * rp) * 128u);
            tma_load_2d(d, &p.tmX, &full[st.s], kb * 64, u * 128);
            for (int g = 0; g < l.n; ++g)
              load_3d<false>(d + 16384 + g * rp * 128, &p.tmA, smem_u32(&full[st.s]), kb * 64, 0, l.ids[g]);
            st.advance(p.tstages);
            ++issued;
          }
          mbar_arrive(&list_empty[li.s]);
          li.advance(kLists);
        }
      if (!ok) {  // leave no copy in flight behind
        *abort_flag = 1;
        for (unsigned i = 0; i < min(issued, (unsigned)p.tstages); ++i) {
          st.back(p.tstages);
          mbar_wait(&full[st.s], st.ph, p.err, DEVERR_WAIT_TMA);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      Ring st, li, ac;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < tiles; u += gridDim.x)
        for (bool more = true; ok && more;) {
          if (!(ok = wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_MMA))) break;
          const int n = lists[li.s].n;
          more = lists[li.s].more;
          mbar_arrive(&list_empty[li.s]);
          li.advance(kLists);
          if (!n) continue;
          ok = wait_on<false>(&d_empty[ac.s], ac.ph ^ 1, abort_flag, p.err, DEVERR_WAIT_MMA);
          const uint32_t d = tmem + ac.s * 256, id = idesc_f16(128, 0, BF16) | ((uint32_t)(n * rp >> 3) << 17);
          for (int kb = 0; ok && kb < nk; ++kb) {
            if (!(ok = wait_on<false>(&full[st.s], st.ph, abort_flag, p.err, DEVERR_WAIT_MMA))) break;
            tc_fence_after();
            const uint64_t x = kdesc(smem_u32(sStage + st.s * p.tstage_bytes)), w = x + (16384 >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f16(d, x + 2 * k, w + 2 * k, id, (kb | k) != 0);
            umma_commit(&empty[st.s]);
            st.advance(p.tstages);
          }
          if (ok) umma_commit(&d_full[ac.s]);
          ac.advance(2);
        }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 2) {
    Ring li;
    bool ok = true;
    int rows[4];
    rows_of<4>(p, blockIdx.x * 128, lane, rows);
    for (int u = blockIdx.x; ok && u < tiles; u += gridDim.x)
      ok = list_adapters<4>(p, u + (int)gridDim.x < tiles ? (u + (int)gridDim.x) * 128 : -1, rows, p.tslots, lists,
                            list_full, list_empty, li, abort_flag, lane);
    if (!ok) *abort_flag = 1;
  } else if (warp >= 4) {
    const int q = warp & 3;
    const int half = p.r <= 32 ? 32 : 64;
    Ring li, ac;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < tiles; u += gridDim.x) {
      const int m = u * 128 + q * 32 + lane;
      for (bool more = true; ok && more;) {
        ok = wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_EPI);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        const SlotList& l = lists[li.s];
        const int n = l.n;
        more = l.more;
        if (n) {
          ok = wait_on<false>(&d_full[ac.s], ac.ph, abort_flag, p.err, DEVERR_WAIT_EPI);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc_fence_after();
          const uint32_t d = tmem + ac.s * 256 + (static_cast<uint32_t>(q * 32) << 16);
          for (int g = 0; g < n; ++g) {
            const uint32_t others = l.others[g][q];
            if (others == 0xffffffffu) continue;  // none of this warp's rows
            const bool mine = m < p.M && !((others >> lane) & 1);
            const float sc = __ldg(p.scale + l.ids[g]);
            for (int c = 0; c < rp; c += 16) {
              uint32_t r[16];
              tmem_ld16(d + g * rp + c, r);
              tmem_wait_ld();
              if (mine) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float x = sc * __uint_as_float(r[2 * k]), y = sc * __uint_as_float(r[2 * k + 1]);
                  hi[k] = pack2<BF16>(x, y);
                  const float2 h = unpack2<BF16>(hi[k]);
                  // a part that is not finite stands alone (inf - inf would be NaN)
                  lo[k] = pack2<BF16>(isinf(h.x) ? 0.f : x - h.x, isinf(h.y) ? 0.f : y - h.y);
                }
                uint4* t = reinterpret_cast<uint4*>(p.T16 + (long long)m * p.t_ld + c / half * (2 * half) + c % half);
                t[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                t[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                t[half / 8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                t[half / 8 + 1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&d_empty[ac.s]);
          ac.advance(2);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&list_empty[li.s]);
        li.advance(kLists);
      }
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- tiles: Y ----

// Out of the way of the epilogue's instructions: the rows of `bad` of a 32 x 32 chunk again, X[m] . W[n] + T[m] . B[a][n] from
// each row's own terms; lane `row` holds row m0 + row as pairs of columns.  One request's activations may be NaN
// in every one of its rows, so 16 rows and columns are taken at a time with mma.sync, where a row's infinities and NaNs
// stay in it; an adapter's product goes to the rows that name it.
template <bool BF16>
__device__ __noinline__ void own_rows(const LoraParams& p, unsigned bad, int m0, int n0, int lane, uint64_t* v) {
  // A lane's 16-byte loads of 8 consecutive k stand for two 16-wide MMA steps: both operands use the same order of k.
  const int at = (lane & 3) * 8;
  auto add = [](float (&d)[2][4], const uint4& a0, const uint4& a1, const uint4& b0, const uint4& b1) {
    const uint32_t f0[4] = {a0.x, a1.x, a0.y, a1.y}, f1[4] = {a0.z, a1.z, a0.w, a1.w};
    mma_16x8x16<BF16>(d[0], f0, b0.x, b0.y);
    mma_16x8x16<BF16>(d[1], f0, b1.x, b1.y);
    mma_16x8x16<BF16>(d[0], f1, b0.z, b0.w);
    mma_16x8x16<BF16>(d[1], f1, b1.z, b1.w);
  };
  auto load = [](const uint16_t* q) { return *reinterpret_cast<const uint4*>(q); };
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    const int mq = m0 + q / 2 * 16, nq = n0 + q % 2 * 16;
    unsigned left = (bad >> q / 2 * 16) & 0xffffu;
    if (!left || nq >= p.N) continue;
    const int r0 = min(mq + lane / 4, p.M - 1), r1 = min(mq + 8 + lane / 4, p.M - 1);  // rows past the last are not stored
    const long long n = nq + lane / 4;                                                // and 8 on: N is a multiple of 16
    float acc[2][4] = {};
    const uint16_t* x0 = static_cast<const uint16_t*>(p.X) + r0 * p.ldx + at;
    const uint16_t* x1 = static_cast<const uint16_t*>(p.X) + r1 * p.ldx + at;
    const uint16_t* w0 = static_cast<const uint16_t*>(p.W) + n * p.K + at;
    const uint16_t* w1 = w0 + 8ll * p.K;
#pragma unroll 2
    for (int k = 0; k < p.K; k += 32) add(acc, load(x0 + k), load(x1 + k), load(w0 + k), load(w1 + k));
    const int half = p.r <= 32 ? 32 : 64, a0 = __ldg(p.rows + r0), a1 = __ldg(p.rows + r1);
    const int mine = __ldg(p.rows + min(mq + (lane & 15), p.M - 1));
    while (left) {  // one adapter of these rows at a time
      const int a = __shfl_sync(0xffffffffu, mine, __ffs(left) - 1);
      left &= ~__ballot_sync(0xffffffffu, mine == a);
      if (a < 0 || a >= p.L) continue;
      float own[2][4] = {}, low[2][4] = {};  // of T's hi and lo parts
      const uint16_t* b0 = static_cast<const uint16_t*>(p.B) + ((long long)a * p.N + n) * p.r;
#pragma unroll 1
      for (int j = at; j < (p.r + 31) / 32 * 32; j += 32) {
        const uint4 none = make_uint4(0, 0, 0, 0);
        const bool in = j < p.r;
        const int col = j / half * (2 * half) + j % half;  // the hi parts of ranks j.., the lo parts `half` on
        const uint16_t *t0 = p.T16 + (long long)r0 * p.t_ld + col, *t1 = p.T16 + (long long)r1 * p.t_ld + col;
        const uint4 bj = in ? load(b0 + j) : none, bk = in ? load(b0 + 8 * p.r + j) : none;
        add(own, in ? load(t0) : none, in ? load(t1) : none, bj, bk);
        add(low, in ? load(t0 + half) : none, in ? load(t1 + half) : none, bj, bk);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)  // an infinity of the hi parts stands: a lo part of zero or of the other sign would make it NaN
          if ((i < 2 ? a0 : a1) == a) acc[c][i] += isinf(own[c][i]) ? own[c][i] : own[c][i] + low[c][i];
    }
    // d[0..1]: row lane / 4, columns 2 (lane & 3) + {0, 1} of 8; d[2..3]: row + 8
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int from = (lane & 7) * 4 + (e & 3);
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = __shfl_sync(0xffffffffu, acc[e / 4][i], from);
      if ((bad >> lane) & 1 && lane / 16 == q / 2) v[q % 2 * 8 + e] = lane & 8 ? f2_pack(t[2], t[3]) : f2_pack(t[0], t[1]);
    }
  }
}

template <bool BF16, bool PAIR>
__global__ void __launch_bounds__(kLThreads, 1) lora_tile_kernel(const __grid_constant__ LoraParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sStage = smem;                            // [stages]: 128 rows of X or T, then rows of W or B, 128 bytes each
  uint8_t* sSlab = smem + p.stages * p.stage_bytes;  // [kEpi][kSlabs], with a residual
  float* sBias = reinterpret_cast<float*>(sSlab + (p.R ? kEpi * kSlabs * kSlab : 0));  // [kEpi][2][32]
  SlotList* lists = reinterpret_cast<SlotList*>(sBias + kEpi * 64);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(lists) + kListBytes);  // [kMaxStages]
  uint64_t* empty = full + kMaxStages;         // [kMaxStages]
  uint64_t* t_full = empty + kMaxStages;       // [kMaxStages] this CTA's T rows landed
  uint64_t* t_clean = t_full + kMaxStages;     // [kMaxStages] other adapters' rows zeroed (a pair: both CTAs', on the first's)
  uint64_t* list_full = t_clean + kMaxStages;  // [kLists]
  uint64_t* list_empty = list_full + kLists;   // [kLists]
  uint64_t* d_full = list_empty + kLists;      // [2] accumulator complete
  uint64_t* d_empty = d_full + 2;              // [2] accumulator read (a pair: by both, on the first CTA's)
  uint64_t* r_full = d_empty + 2;              // [kEpi][kSlabs] residual landed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(r_full + kEpi * kSlabs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int first = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x, step = PAIR ? (int)gridDim.x / 2 : (int)gridDim.x;
  const bool issues = rank == 0;  // this CTA's warp 1 issues the MMAs
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&t_full[i], 1);
      mbar_init(&t_clean[i], PAIR ? 2 : 1);
    }
    // readers of a list entry: loads, MMAs (where they are issued), zeroing, epilogue
    for (int i = 0; i < kLists; ++i) { mbar_init(&list_full[i], 1); mbar_init(&list_empty[i], (issues ? 3 : 2) + kEpi); }
    for (int i = 0; i < 2; ++i) { mbar_init(&d_full[i], 1); mbar_init(&d_empty[i], (PAIR ? 2 : 1) * kEpi); }
    for (int i = 0; i < kEpi * kSlabs; ++i) mbar_init(&r_full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
    else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  }
  tc_fence_before();
  if (PAIR) cluster_sync();  // both CTAs' barriers are initialised before either signals the other
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t full0 = PAIR ? mapa_shared(smem_u32(full), 0) : smem_u32(full);
  const uint32_t t_clean0 = PAIR ? mapa_shared(smem_u32(t_clean), 0) : smem_u32(t_clean);
  const uint32_t d_empty0 = PAIR ? mapa_shared(smem_u32(d_empty), 0) : smem_u32(d_empty);
  pdl_trigger();
  // lora_t_kernel let this one start after its own wait for earlier kernels: X, W, the indices, R and Y are safe to use
  // at once, T only after pdl_wait.
  constexpr int TM = PAIR ? 256 : 128;
  const int units = p.mt * p.nt, nk = p.K / 64;
  const int groups = p.r <= 32 ? 1 : (p.r + 63) / 64;  // rank groups, each one block of B
  const uint32_t b_rows = PAIR ? p.BN / 2 : p.BN;      // rows of W or B that this CTA loads

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tmX);
      tma_prefetch_desc(&p.tmW);
      tma_prefetch_desc(&p.tmT);
      tma_prefetch_desc(&p.tmB);
      Ring st, li;
      bool ok = true, waited = false;
      unsigned issued = 0, t_any = 0, t_ph = 0;  // t_ph: phase that the last T copy into a stage completes
      auto load_t = [&](int col, int m0) {
        t_ph ^= ((t_any >> st.s) & 1) << st.s;
        t_any |= 1u << st.s;
        mbar_arrive_expect_tx(&t_full[st.s], 16384u);
        tma_load_2d(sStage + st.s * p.stage_bytes, &p.tmT, &t_full[st.s], col, m0);
      };
      auto stage = [&](uint32_t bytes) {  // the next free stage, armed for `bytes` of each CTA
        if (!wait_on<PAIR>(&empty[st.s], st.ph ^ 1, abort_flag, p.err, DEVERR_WAIT_TMA)) return false;
        if (issues) mbar_arrive_expect_tx(&full[st.s], PAIR ? 2 * bytes : bytes);  // 0: nothing but T, on t_full
        ++issued;
        return true;
      };
      for (int u = first; ok && u < units; u += step) {
        const int m0 = u / p.nt * TM + rank * 128, n0 = u % p.nt * p.BN + rank * (int)b_rows;
        for (int kb = 0; ok && kb < nk; ++kb) {
          if (!(ok = stage(16384u + b_rows * 128u))) break;
          uint8_t* d = sStage + st.s * p.stage_bytes;
          load_2d<PAIR>(d, &p.tmX, full0 + st.s * 8, kb * 64, m0);
          load_2d<PAIR>(d + 16384, &p.tmW, full0 + st.s * 8, kb * 64, n0);
          st.advance(p.stages);
        }
        for (bool more = true; ok && more;) {
          if (!(ok = wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_TMA))) break;
          const SlotList& l = lists[li.s];
          more = l.more;
          if (l.n && !waited) {
            pdl_wait();
            waited = true;
          }
          for (int g = 0; ok && g < l.n; ++g)
            for (int c = 0; ok && c < groups; ++c) {
              if (!(ok = stage(b_rows * 128u))) break;
              uint8_t* d = sStage + st.s * p.stage_bytes;
              load_t(c * 128, m0);
              load_3d<PAIR>(d + 16384, &p.tmB, full0 + st.s * 8, c * 64, n0, l.ids[g]);
              st.advance(p.stages);
              if (p.r > 32) {  // the lo parts, against the same B
                if (!(ok = stage(0u))) break;
                load_t(c * 128 + 64, m0);
                st.advance(p.stages);
              }
            }
          mbar_arrive(&list_empty[li.s]);
          li.advance(kLists);
        }
      }
      if (!ok) {  // leave no copy in flight behind
        *abort_flag = 1;
        for (unsigned i = 0; issues && i < min(issued, (unsigned)p.stages); ++i) {
          st.back(p.stages);
          mbar_wait<PAIR>(&full[st.s], st.ph, p.err, DEVERR_WAIT_TMA);
        }
        for (int i = 0; i < p.stages; ++i)
          if ((t_any >> i) & 1) mbar_wait(&t_full[i], (t_ph >> i) & 1, p.err, DEVERR_WAIT_TMA);
      }
    }
  } else if (warp == 1) {
    if (issues && elect_one()) {
      Ring st, li;
      bool ok = true;
      int nu = 0;
      const uint32_t id = idesc_f16(TM, 0, BF16) | ((uint32_t)(p.BN >> 3) << 17);
      auto commit = [&](uint64_t* bar) {
        if (PAIR) umma_commit_pair(bar, 0x3);
        else umma_commit(bar);
      };
      auto stage = [&]() {
        const bool r = wait_on<PAIR>(&full[st.s], st.ph, abort_flag, p.err, DEVERR_WAIT_MMA);
        tc_fence_after();
        return r;
      };
      unsigned ph_c = 0;  // phases of t_clean, one bit per stage
      auto t_stage = [&]() {
        if (!stage()) return false;
        const bool r = wait_on<PAIR>(&t_clean[st.s], (ph_c >> st.s) & 1, abort_flag, p.err, DEVERR_WAIT_MMA);
        ph_c ^= 1u << st.s;
        tc_fence_after();
        return r;
      };
      auto add = [&](uint32_t d, uint64_t a, uint64_t b) {
        if (PAIR) umma_f16_pair(d, a, b, id, 1);
        else umma_f16(d, a, b, id, 1);
      };
      for (int u = first; ok && u < units; u += step, ++nu) {
        const int ab = nu & 1;
        const uint32_t d = tmem + ab * 256;
        ok = wait_on<PAIR>(&d_empty[ab], ((nu >> 1) & 1) ^ 1, abort_flag, p.err, DEVERR_WAIT_MMA);
        for (int kb = 0; ok && kb < nk; ++kb) {
          if (!(ok = stage())) break;
          const uint64_t ad = kdesc(smem_u32(sStage + st.s * p.stage_bytes)), bd = ad + (16384 >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (PAIR) umma_f16_pair(d, ad + 2 * k, bd + 2 * k, id, (kb | k) != 0);
            else umma_f16(d, ad + 2 * k, bd + 2 * k, id, (kb | k) != 0);
          }
          commit(&empty[st.s]);
          st.advance(p.stages);
        }
        for (bool more = true; ok && more;) {
          if (!(ok = wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_MMA))) break;
          const SlotList& l = lists[li.s];
          more = l.more;
          const int n = l.n;
          for (int g = 0; ok && g < n; ++g)
            for (int c = 0; ok && c < groups; ++c) {
              const int steps = (min(p.r - c * 64, 64) + 15) / 16;
              if (!(ok = t_stage())) break;
              const uint64_t hi = kdesc(smem_u32(sStage + st.s * p.stage_bytes)), bd = hi + (16384 >> 4);
              const int s0 = st.s;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < steps) add(d, hi + 2 * k, bd + 2 * k);
              st.advance(p.stages);
              uint64_t lo = hi + 4;  // r <= 32: the same block's second half
              if (p.r > 32) {
                if (!(ok = t_stage())) break;
                lo = kdesc(smem_u32(sStage + st.s * p.stage_bytes));
              }
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < steps) add(d, lo + 2 * k, bd + 2 * k);
              commit(&empty[s0]);
              if (p.r > 32) {
                commit(&empty[st.s]);
                st.advance(p.stages);
              }
            }
          mbar_arrive(&list_empty[li.s]);
          li.advance(kLists);
        }
        if (ok) commit(&d_full[ab]);
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 2) {
    Ring li;
    bool ok = true;
    int rows[TM / 32];
    rows_of<TM / 32>(p, first / p.nt * TM, lane, rows);
    for (int u = first; ok && u < units; u += step)
      ok = list_adapters<TM / 32>(p, u + step < units ? (u + step) / p.nt * TM : -1, rows, kSlots, lists, list_full,
                                  list_empty, li, abort_flag, lane);
    if (!ok) *abort_flag = 1;
  } else if (warp == 3) {
    Ring st, li;
    unsigned ph = 0;  // phases of t_full
    bool ok = true;
    for (int u = first; ok && u < units; u += step) {
      for (int kb = 0; kb < nk; ++kb) st.advance(p.stages);
      for (bool more = true; ok && more;) {
        ok = __all_sync(0xffffffffu, wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_EPI));
        if (!ok) break;
        const SlotList& l = lists[li.s];
        const int n = l.n;
        more = l.more;
        for (int g = 0; ok && g < n; ++g) {
          uint32_t others[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) others[i] = l.others[g][rank * 4 + i];
          for (int c = 0; ok && c < groups * (p.r <= 32 ? 1 : 2); ++c) {
            ok = __all_sync(0xffffffffu, wait_on<false>(&t_full[st.s], (ph >> st.s) & 1, abort_flag, p.err, DEVERR_WAIT_EPI));
            if (!ok) break;
            ph ^= 1u << st.s;
            if (others[0] | others[1] | others[2] | others[3]) {
              // a warp's stores cover four whole rows: lane / 8 the row, lane % 8 its 16-byte piece
              uint4* t = reinterpret_cast<uint4*>(sStage + st.s * p.stage_bytes);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (others[i]) {  // warp-uniform
#pragma unroll
                  for (int k = 0; k < 8; ++k)
                    if ((others[i] >> (k * 4 + lane / 8)) & 1) t[(i * 32 + k * 4) * 8 + lane] = make_uint4(0, 0, 0, 0);
                }
              fence_async_smem();
              __syncwarp();
            }
            if (lane == 0) {
              if (PAIR) mbar_arrive_cluster(t_clean0 + st.s * 8);
              else mbar_arrive(&t_clean[st.s]);
            }
            st.advance(p.stages);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&list_empty[li.s]);
        li.advance(kLists);
      }
    }
    if (!ok) *abort_flag = 1;
  } else {
    const int ew = warp - 4, q = warp & 3, part = ew / 4;
    uint8_t* slabs = sSlab + ew * kSlabs * kSlab;
    uint64_t* rb = r_full + ew * kSlabs;
    float* bs = sBias + ew * 64;
    // The warp's chunks (32 rows by 32 columns, columns part, part + kEpiPer, ... of each tile), as one sequence over its
    // tiles: residual and bias are fetched one chunk ahead.
    struct Chunk {
      int u, i, mine, m0, n0;  // tile, chunk, chunks of the tile; first row of the warp, first column of the tile
    };
    const int dm = step / p.nt * TM, dn = step % p.nt * p.BN, n_end = p.nt * p.BN;
    auto chunks_of = [&](Chunk& c) {
      c.i = 0;
      c.mine = c.m0 < p.M ? ((min(p.BN, p.N - c.n0) + 31) / 32 - part + kEpiPer - 1) / kEpiPer : 0;
    };
    auto next_tile = [&](Chunk& c) {
      c.u += step;
      c.m0 += dm;
      c.n0 += dn;
      if (c.n0 >= n_end) { c.n0 -= n_end; c.m0 += TM; }
      chunks_of(c);
    };
    auto to_chunk = [&](Chunk& c) {  // on to the next tile while this one has no more chunks
      while (c.u < units && c.i >= c.mine) next_tile(c);
    };
    auto column = [&](const Chunk& c) { return c.n0 + (part + kEpiPer * c.i) * 32; };
    Chunk c, f;  // this chunk, the next one
    c.u = first;
    c.m0 = first / p.nt * TM + rank * 128 + q * 32;
    c.n0 = first % p.nt * p.BN;
    chunks_of(c);
    f = c;
    to_chunk(f);
    unsigned k = 0, fetched = 0, r_ph = 0;  // chunks so far, residuals fetched, phases of their barriers
    float bias = 0.f;                       // of the next chunk
    auto fetch = [&] {
      if (f.u >= units) return;
      const int n = column(f);
      if (p.bias) bias = n + lane < p.N ? __ldg(p.bias + n + lane) : 0.f;
      if (p.R) {
        const int sl = fetched++ % kSlabs;
        if (lane == 0) {
          mbar_arrive_expect_tx(&rb[sl], kSlab);
          tma_load_2d(slabs + sl * kSlab, &p.tmR, &rb[sl], n, f.m0);
        }
      }
      ++f.i;
      to_chunk(f);
    };
    Ring li;
    bool ok = true;
    int nu = 0;
    fetch();
    pdl_wait();  // this grid is not over before lora_t_kernel is
    for (; ok && c.u < units; next_tile(c), ++nu) {
      const int ab = nu & 1;
      bool mixed = false;  // some of the tile's rows do not take its first adapter
      for (bool more = true; ok && more;) {
        ok = __all_sync(0xffffffffu, wait_on<false>(&list_full[li.s], li.ph, abort_flag, p.err, DEVERR_WAIT_EPI));
        if (!ok) break;
        const SlotList& l = lists[li.s];
        more = l.more;
        mixed = mixed || l.n > 1 || more || (l.n && __any_sync(0xffffffffu, lane < TM / 32 && l.others[0][lane % 8]));
        __syncwarp();
        if (lane == 0) mbar_arrive(&list_empty[li.s]);
        li.advance(kLists);
      }
      ok = ok && wait_on<PAIR>(&d_full[ab], (nu >> 1) & 1, abort_flag, p.err, DEVERR_WAIT_EPI);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + ab * 256 + part * 32 + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (; c.i < c.mine; ++c.i, ++k) {
        const int nb = column(c), m = c.m0 + lane;
        float* bk = bs + (k & 1) * 32;
        uint32_t r[32];
        tmem_ld32(d + c.i * 32 * kEpiPer, r);
        if (p.bias) bk[lane] = bias;
        __syncwarp();
        fetch();  // into the slab that the chunk before this one has read
        tmem_wait_ld();
        uint64_t v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = f2_pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
        if (mixed) {
          uint64_t z = 0;
#pragma unroll
          for (int e = 0; e < 16; ++e) z = fma2(v[e], 0, z);  // NaN if any value is not finite
          const unsigned bad = __ballot_sync(0xffffffffu, lo_f(z) + hi_f(z) != 0.f && c.m0 + lane < p.M);
          if (bad) {
            uint64_t t[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) t[e] = v[e];
            own_rows<BF16>(p, bad, c.m0, nb, lane, t);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = t[e];
          }
        }
        if (p.bias) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const ulonglong2 t = reinterpret_cast<const ulonglong2*>(bk)[e];
            v[2 * e] = add2(v[2 * e], t.x);
            v[2 * e + 1] = add2(v[2 * e + 1], t.y);
          }
        }
        if (p.act == 1) {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = f2_pack(silu_fast(lo_f(v[e])), silu_fast(hi_f(v[e])));
        } else if (p.act == 2) {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = gelu2(v[e]);
        }
        if (p.R) {
          const int sl = k % kSlabs;
          ok = __all_sync(0xffffffffu, wait_on<false>(&rb[sl], (r_ph >> sl) & 1, abort_flag, p.err, DEVERR_WAIT_EPI));
          if (!ok) break;  // the slab is not there: the copy is waited for once more below
          r_ph ^= 1u << sl;
          const uint4* rp = reinterpret_cast<const uint4*>(slabs + sl * kSlab + lane * 64);  // 64-byte rows, 64-byte swizzle
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 t = rp[e ^ ((lane >> 1) & 3)];
            const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float2 g = unpack2<BF16>(w[x]);
              v[4 * e + x] = add2(v[4 * e + x], f2_pack(g.x, g.y));
            }
          }
        }
        if (m < p.M) {
          uint16_t* dst = static_cast<uint16_t*>(p.Y) + m * p.ldy + nb;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (nb + 16 * h < p.N) {
              uint32_t t[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) t[e] = pack2<BF16>(lo_f(v[8 * h + e]), hi_f(v[8 * h + e]));
              if (p.wide)
                asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + 16 * h), "r"(t[0]), "r"(t[1]),
                             "r"(t[2]), "r"(t[3]), "r"(t[4]), "r"(t[5]), "r"(t[6]), "r"(t[7])
                             : "memory");
              else
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  reinterpret_cast<uint4*>(dst)[2 * h + e] = make_uint4(t[4 * e], t[4 * e + 1], t[4 * e + 2], t[4 * e + 3]);
            }
        }
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        // the reads are complete (tcgen05.wait): nothing else is handed over, so no release
        if (PAIR)
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(d_empty0 + ab * 8) : "memory");
        else
          mbar_arrive(&d_empty[ab]);
      }
    }
    if (!ok) *abort_flag = 1;
    for (; p.R && k < fetched; ++k) {  // only after giving up: residuals still on their way
      mbar_wait(&rb[k % kSlabs], (r_ph >> (k % kSlabs)) & 1, p.err, DEVERR_WAIT_EPI);
      r_ph ^= 1u << (k % kSlabs);
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// ---- few rows ----

// s[j] = x . w[j] over K values by one warp, for J rows of w that lie K apart; every lane gets them.
template <bool BF16, int J>
__device__ __forceinline__ void dot_k(const uint16_t* x, const uint16_t* w, int K, int lane, float (&s)[J]) {
#pragma unroll
  for (int j = 0; j < J; ++j) s[j] = 0.f;
#pragma unroll(4 / J)
  for (int k = lane * 8; k < K; k += 256) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + k));
    uint4 v[J];
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = __ldg(reinterpret_cast<const uint4*>(w + (long long)j * K + k));
    const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t vv[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<BF16>(uu[e]), g = unpack2<BF16>(vv[e]);
        s[j] = fmaf(f.x, g.x, fmaf(f.y, g.y, s[j]));
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
}

// T[m][j] = scale[a] * X[m] . A[a][j]: one warp per value, eight of one row to a block.
template <bool BF16>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const __grid_constant__ LoraParams p) {
  pdl_begin();
  const int m = blockIdx.y, j = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x & 31;
  int a = __ldg(p.rows + m);
  if (a >= p.L) {
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.err, DEVERR_BOUNDS);
    a = -1;
  }
  if (a < 0) return;  // nothing reads this row of T
  float s[1];
  dot_k<BF16>(static_cast<const uint16_t*>(p.X) + m * p.ldx, static_cast<const uint16_t*>(p.A) + ((long long)a * p.r + j) * p.K,
              p.K, lane, s);
  if (lane == 0) p.T[m * p.r + j] = __ldg(p.scale + a) * s[0];
}

// 16 NT columns of Y for 8 MT rows per block.  The 8 warps take shares of K (32-wide blocks in turn), summed in shared
// memory.  A lane's 16-byte loads of 8 consecutive k stand for two 16-wide MMA steps: both
// operands use the same order of k.  Bound: the bytes of W and B, and from L2 those of X, which every block reads whole.
// CLUSTER: no first launch; the eight blocks of a cluster share out the values of T, which eight more warps of each compute
// and hand to all through distributed shared memory while the MMAs run.
template <bool BF16, int MT, bool CLUSTER, int NT = 1>
__global__ void __launch_bounds__(CLUSTER ? 512 : 256) lora_skinny_kernel(const __grid_constant__ LoraParams p) {
  constexpr int KW = 8, ROWS = 8 * MT, COLS = 16 * NT, AHEAD = 8, RANK = NT > 1 ? 64 : 128;
  __shared__ float red[KW][ROWS][COLS + 1];
  __shared__ __align__(16) float ts[ROWS * RANK];  // T of the rows
  __shared__ int as[ROWS];                                         // their adapters
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * COLS, m0 = blockIdx.y * ROWS;
  constexpr int THREADS = CLUSTER ? 512 : 256;
  if (CLUSTER) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // 1: this block has started
    pdl_wait();
  }
  // The shrink kernel lets this one start after its own wait for earlier kernels: X, W, B and the indices may be read at
  // once, T, R and Y only after it.
  pdl_trigger();
  for (int i = threadIdx.x; i < ROWS; i += THREADS) {
    int a = m0 + i < p.M ? __ldg(p.rows + m0 + i) : -1;
    if (a >= p.L) {
      if (CLUSTER && blockIdx.x == 0) atomicOr(p.err, DEVERR_BOUNDS);
      a = -1;
    }
    as[i] = a;
  }
  if (CLUSTER && warp >= 8) {
    const int n = min(ROWS, p.M - m0) * p.r;
    bool waited = false;
    constexpr int J = 2;  // values of a row at a time
    for (int v = ((int)cluster_ctarank() + 8 * (warp - 8)) * J; v < n; v += 64 * J) {
      const int m = v / p.r, a = __ldg(p.rows + m0 + m);
      float s[J] = {};
      if (a >= 0 && a < p.L) {
        dot_k<BF16>(static_cast<const uint16_t*>(p.X) + (m0 + m) * p.ldx,
                    static_cast<const uint16_t*>(p.A) + ((long long)a * p.r + v % p.r) * p.K, p.K, lane, s);
#pragma unroll
        for (int j = 0; j < J; ++j) s[j] *= __ldg(p.scale + a);
      }
      if (!waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // 1: all eight have started
      waited = true;
      if (lane < 8) {
        const uint32_t d = mapa_shared(smem_u32(ts + v), lane);
#pragma unroll
        for (int j = 0; j < J; ++j) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(d + 4 * j), "f"(s[j]) : "memory");
      }
    }
    if (!waited) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
  const int kw = warp;
  float acc[NT][MT][4] = {};
  const uint16_t* wp[2 * NT];
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i)
    wp[i] = static_cast<const uint16_t*>(p.W) + (long long)min(n0 + i * 8 + lane / 4, p.N - 1) * p.K + (lane & 3) * 8;
  const uint16_t* xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)  // rows and columns past the last are computed and not stored
    xp[t] = static_cast<const uint16_t*>(p.X) + min(m0 + t * 8 + lane / 4, p.M - 1) * p.ldx + (lane & 3) * 8;
#pragma unroll (NT > 1 ? 2 : 4)
  for (int k = kw * 32; k < p.K; k += KW * 32) {
    uint4 a[2 * NT], b[MT];
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) a[i] = __ldg(reinterpret_cast<const uint4*>(wp[i] + k));
#pragma unroll
    for (int t = 0; t < MT; ++t) b[t] = __ldg(reinterpret_cast<const uint4*>(xp[t] + k));
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      const uint4 a0 = a[2 * c], a1 = a[2 * c + 1];
      const uint32_t f0[4] = {a0.x, a1.x, a0.y, a1.y}, f1[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        mma_16x8x16<BF16>(acc[c][t], f0, b[t].x, b[t].y);
        mma_16x8x16<BF16>(acc[c][t], f1, b[t].z, b[t].w);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int t = 0; t < MT; ++t) {  // d[0..1]: column lane / 4, rows 2 (lane & 3) + {0, 1}; d[2..3]: column + 8
      const int m = t * 8 + (lane & 3) * 2, n = c * 16 + lane / 4;
      red[kw][m][n] = acc[c][t][0];
      red[kw][m + 1][n] = acc[c][t][1];
      red[kw][m][n + 8] = acc[c][t][2];
      red[kw][m + 1][n + 8] = acc[c][t][3];
    }
  if (CLUSTER) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // 1
  }
  if (CLUSTER) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // 2: this warp's values of T are written
  __syncthreads();
  // One output per thread at a time, neighbours in a row: its B row in pieces of AHEAD x 16 bytes, the next piece (of this
  // output or of the thread's next one) already on its way.
  constexpr int total = ROWS * COLS;
  uint4 u[AHEAD];
  auto b_row = [&](int o) -> const uint4* {  // null: no adapter, or outside Y
    const int n = n0 + o % COLS, a = o < total ? as[o / COLS] : -1;
    return a >= 0 && n < p.N ? reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.B) + ((long long)a * p.N + n) * p.r)
                             : nullptr;
  };
  const int pieces = p.r / 8;
  auto fetch = [&](const uint4* row, int c) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) u[i] = row && c + i < pieces ? __ldg(row + c + i) : make_uint4(0, 0, 0, 0);
  };
  const uint4* row = b_row(threadIdx.x);
  fetch(row, 0);
  if (CLUSTER) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    pdl_wait();  // T is complete
  }
  if (!CLUSTER) {
    for (int i = threadIdx.x; i < ROWS * p.r; i += THREADS) ts[i] = m0 * p.r + i < p.M * p.r ? p.T[(long long)m0 * p.r + i] : 0.f;
    __syncthreads();
  }
  for (int o = threadIdx.x; o < total; o += THREADS) {
    const int ml = o / COLS, n = n0 + o % COLS, m = m0 + ml;
    const float4* t = reinterpret_cast<const float4*>(ts + ml * p.r);
    float s = 0.f, s2 = 0.f;
    auto dot = [&](const uint4& v, const float4* t) {
      const float4 ta = t[0], tb = t[1];
      const float2 f0 = unpack2<BF16>(v.x), f1 = unpack2<BF16>(v.y), f2 = unpack2<BF16>(v.z), f3 = unpack2<BF16>(v.w);
      s = fmaf(ta.x, f0.x, fmaf(ta.y, f0.y, fmaf(ta.z, f1.x, fmaf(ta.w, f1.y, s))));
      s2 = fmaf(tb.x, f2.x, fmaf(tb.y, f2.y, fmaf(tb.z, f3.x, fmaf(tb.w, f3.y, s2))));
    };
    const uint4* next = b_row(o + THREADS);
#pragma unroll 1
    for (int c = 0; c < pieces; c += AHEAD) {
      uint4 now[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) now[i] = u[i];
      if (c + AHEAD < pieces) fetch(row, c + AHEAD);
      else fetch(next, 0);
      if (row) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          if (c + i < pieces) dot(now[i], t + 2 * (c + i));
      }
    }
    row = next;
    if (m < p.M && n < p.N) {
#pragma unroll
      for (int x = 0; x < KW; ++x) s += red[x][ml][o % COLS];
      s += s2;
      if (p.bias) s += __ldg(p.bias + n);
      s = act_of(s, p.act);
      if (p.R) s += unpack2<BF16>(static_cast<const uint16_t*>(p.R)[m * p.ldr + n]).x;
      static_cast<uint16_t*>(p.Y)[m * p.ldy + n] = (uint16_t)pack2<BF16>(s, 0.f);
    }
  }
}

// Few rows in one launch: row tiles of 8 per block, or 0 for two launches.  Each cluster of eight blocks (128 columns)
// works out T of its rows itself; up to 12 clusters find room at once (16 took twice the time of 10).  It saves a launch
// and the scratch, 5 us of a caller's time (8 x 1280 x 1280, rank 16: 8.4 us a call against 13.5), and costs the GPU up to 2 us
// at 256 values of T (in a graph, rank 16: 4.5 us against 4.1, rank 32: 6.1 against 4.3; 16 x 640 x 640, rank 16: 3.7 against
// 3.9; with 512 values 9.3 against 5.2).
int one_launch(long long M, long long N, long long r) {
  const long long tiles = (M + 7) / 8, columns = (N + 127) / 128;
  for (int mt = 1; mt <= 4; mt *= 2)
    if (columns * ((tiles + mt - 1) / mt) <= 12) return std::min<long long>(M, 8 * mt) * r <= 256 ? mt : 0;
  return 0;
}

template <bool BF16>
int launch_skinny(Ctx* c, const LoraParams& p) {
  const int tiles = (p.M + 7) / 8;
  if (const int mt = one_launch(p.M, p.N, p.r)) {
    const dim3 grid((p.N + 127) / 128 * 8, (tiles + mt - 1) / mt);
    auto kern = mt == 1 ? lora_skinny_kernel<BF16, 1, true> : mt == 2 ? lora_skinny_kernel<BF16, 2, true> : lora_skinny_kernel<BF16, 4, true>;
    launch_k_cluster(kern, grid, 512, 0, c->stream, 8, p);
    return check_launch(c, "linear_lora");
  }
  launch_k(lora_shrink_kernel<BF16>, dim3(p.r / 8, p.M), 256, 0, c->stream, p);
  const int rc = check_launch(c, "linear_lora");
  if (rc != DI_OK) return rc;
  // Row tiles per block: up to four (eight: 128 x 4096 x 4096 60 us instead of 48), fewer while the blocks are fewer than
  // the SMs.
  int mt = tiles == 1 ? 1 : tiles == 2 ? 2 : 4;
  while (mt > 1 && p.N / 16 * ((tiles + mt - 1) / mt) < c->num_sms) mt /= 2;
  auto go = [&](auto kern, int cols = 16) {
    launch_k(kern, dim3((p.N + cols - 1) / cols, (tiles + mt - 1) / mt), 256, 0, c->stream, p);
  };
  // 32 columns per block where enough blocks remain (and T and the sums fit shared memory): X comes from L2 half as often
  // (64 x 1024 x 4096: 12.7 us, with 16 columns 14.8; 128 x 4096 x 4096: 38.6 and 47.7)
  const bool wide = mt == 4 && p.r <= 64 && (p.N + 31) / 32 * ((tiles + 3) / 4) >= c->num_sms;
  if (mt == 1) go(lora_skinny_kernel<BF16, 1, false>);
  else if (mt == 2) go(lora_skinny_kernel<BF16, 2, false>);
  else if (wide) go(lora_skinny_kernel<BF16, 4, false, 2>, 32);
  else go(lora_skinny_kernel<BF16, 4, false>);
  return check_launch(c, "linear_lora");
}

// CTA pairs that can be resident at once (both SMs of a pair lie in one GPC), per device.
template <bool BF16>
int resident_pairs(Ctx* c) {
  static int known[32] = {};
  int& n = known[c->device & 31];
  if (n) return n;
  int got = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (c->num_sms / 2));
  cfg.blockDim = dim3(kLThreads);
  cfg.dynamicSmemBytes = 232448;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&got, lora_tile_kernel<BF16, true>, &cfg) != cudaSuccess || got < 1) got = c->num_sms / 4;
  cudaGetLastError();
  return n = std::min(got, c->num_sms / 2);
}

template <bool BF16>
int launch_tiles(Ctx* c, LoraParams& p) {
  static unsigned attr_done = 0;
  if (!(attr_done & (1u << (c->device & 31)))) {
    if (cudaFuncSetAttribute(lora_t_kernel<BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess ||
        cudaFuncSetAttribute(lora_tile_kernel<BF16, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess ||
        cudaFuncSetAttribute(lora_tile_kernel<BF16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess)
      return cudaGetLastError(), set_error(c, DI_ECUDA, "linear_lora: shared memory attribute");
    attr_done |= 1u << (c->device & 31);
  }
  // Column width and pairing: a K block takes 2 BN cycles of MMAs or its stage's bytes at some 45 bytes a cycle from L2,
  // whichever is more; a tile's epilogue (about 9 cycles a column and CTA) runs under the next main loop; the last
  // tile's and the first loads do not.
  bool pair = false;
  double best = 1e30;
  const int pairs = resident_pairs<BF16>(c);
  for (int pr = 0; pr < 2; ++pr) {
    const int mt = pr ? (p.M + 255) / 256 : (p.M + 127) / 128;
    for (int bn = 256; bn >= 32; bn -= 32) {
      const int nt = (p.N + bn - 1) / bn, slots = pr ? pairs : c->num_sms;
      const double rounds = (double)(((long long)mt * nt + slots - 1) / slots);
      const double kb = std::max(2.0 * bn, (128 + (pr ? bn / 2 : bn)) * 128 / 45.0);
      const double loop = (p.K / 64 + 1) * kb, epi = 9.0 * bn;
      const double cost = rounds * std::max(loop, epi) + epi + 1500.0;
      if (cost < best * 0.999) {
        best = cost;
        p.BN = bn;
        p.nt = nt;
        p.mt = mt;
        pair = pr != 0;
      }
    }
  }
  const int b_rows = pair ? p.BN / 2 : p.BN;
  p.stage_bytes = (16384 + b_rows * 128 + 1023) / 1024 * 1024;
  const uint32_t fixed = kFixedSmem + (p.R ? kEpi * kSlabs * kSlab : 0);
  p.stages = (int)std::min<uint32_t>(kMaxStages, (232448 - fixed) / p.stage_bytes);
  const uint32_t smem = fixed + p.stages * p.stage_bytes;
  p.wide = (reinterpret_cast<uintptr_t>(p.Y) & 31) == 0 && p.ldy % 16 == 0;
  p.t_ld = p.r <= 32 ? 64 : (p.r + 63) / 64 * 128;
  const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t M = p.M, N = p.N, K = p.K, r = p.r, tl = p.t_ld;
  const uint64_t xd[2] = {K, M}, wd[2] = {K, N}, td[2] = {tl, M}, bd[3] = {r, N, (uint64_t)p.L};
  const uint64_t xs[1] = {(uint64_t)p.ldx * 2}, ws[1] = {K * 2}, ts[1] = {tl * 2}, bs[2] = {r * 2, N * r * 2};
  const uint32_t xb[2] = {64, 128}, wb[2] = {64, (uint32_t)b_rows}, bb[3] = {64, (uint32_t)b_rows, 1};
  const uint64_t rd[2] = {N, M}, rs[1] = {(uint64_t)p.ldr * 2};
  const uint32_t rb[2] = {32, 32};
  std::string err;
  if (!make_tmap(&p.tmX, dt, 2, p.X, xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmW, dt, 2, p.W, wd, ws, wb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmT, dt, 2, p.T16, td, ts, xb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmB, dt, 3, p.B, bd, bs, bb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      (p.R && !make_tmap(&p.tmR, dt, 2, p.R, rd, rs, rb, CU_TENSOR_MAP_SWIZZLE_64B, &err)))
    return set_error(c, DI_EINVAL, "linear_lora: " + err);
  const int rp = (p.r + 15) / 16 * 16;
  p.tslots = std::max(1, std::min({p.L, kSlots, 256 / rp}));
  p.tstage_bytes = 16384 + p.tslots * rp * 128;
  p.tstages = (int)std::min<uint32_t>(5, (232448 - kTFixedSmem) / p.tstage_bytes);
  const uint64_t ad[3] = {K, r, (uint64_t)p.L}, as[2] = {K * 2, r * K * 2};
  const uint32_t ab[3] = {64, (uint32_t)rp, 1};
  if (!make_tmap(&p.tmA, dt, 3, p.A, ad, as, ab, CU_TENSOR_MAP_SWIZZLE_128B, &err))
    return set_error(c, DI_EINVAL, "linear_lora: " + err);
  launch_k(lora_t_kernel<BF16>, dim3((unsigned)std::min<long long>((p.M + 127LL) / 128, c->num_sms)), dim3(kTThreads),
           kTFixedSmem + p.tstages * p.tstage_bytes, c->stream, p);
  const int rc = check_launch(c, "linear_lora");
  if (rc != DI_OK) return rc;
  const long long units = (long long)p.mt * p.nt;
  if (pair)
    launch_k_cluster(lora_tile_kernel<BF16, true>, dim3(2 * (unsigned)std::min<long long>(units, pairs)), dim3(kLThreads), smem,
                     c->stream, 2, p);
  else
    launch_k(lora_tile_kernel<BF16, false>, dim3((unsigned)std::min<long long>(units, c->num_sms)), dim3(kLThreads), smem,
             c->stream, p);
  return check_launch(c, "linear_lora");
}

}  // namespace
}  // namespace di

using namespace di;

namespace {
bool fits_int(const long long* v, int n) {
  for (int i = 0; i < n; ++i)
    if (v[i] < 0 || v[i] > (1ll << 30)) return false;
  return true;
}
}  // namespace

extern "C" size_t di_linear_lora_workspace(di_ctx_t h, const long long cfg[9]) {
  if (!h || !cfg || !fits_int(cfg, 5)) return 0;
  const size_t M = cfg[0], rank = cfg[3];
  if (M <= (size_t)kSkinnyRows) return one_launch(cfg[0], cfg[1], cfg[3]) ? 0 : M * rank * 4;
  return M * (rank <= 32 ? 64 : (rank + 63) / 64 * 128) * 2;
}

extern "C" int di_linear_lora(di_ctx_t h, int dtype, const long long cfg[9], const void* X, const void* W, const void* A,
                              const void* B, const float* scale, const int* row_adapter, const float* bias, const void* R,
                              void* Y, void* ws, size_t ws_bytes) {
  Ctx* c = ctx_of(h);
  if (!c || (dtype != DI_F16 && dtype != DI_BF16)) return DI_EINVAL;
  DeviceGuard guard(c->device);
  if (!cfg || !fits_int(cfg, 5) || !X || !W || !A || !B || !scale || !row_adapter || !Y)
    return set_error(c, DI_EINVAL, "linear_lora: bad shape or missing tensor");
  const int M = (int)cfg[0], N = (int)cfg[1], K = (int)cfg[2], rank = (int)cfg[3], L = (int)cfg[4];
  const long long ldx = cfg[5], ldr = cfg[6], ldy = cfg[7], act = cfg[8];
  if (M <= 0 || N <= 0 || K <= 0 || L <= 0) return set_error(c, DI_EINVAL, "linear_lora: bad shape or missing tensor");
  if (K % 64 || N % 16) return set_error(c, DI_EUNSUPPORTED, "linear_lora: K must be a multiple of 64, N of 16");
  if (rank < 8 || rank > 128 || rank % 8)
    return set_error(c, DI_EUNSUPPORTED, "linear_lora: the rank must be a multiple of 8, 8 to 128");
  if (act < 0 || act > 2) return set_error(c, DI_EINVAL, "linear_lora: act must be 0 (none), 1 (SiLU) or 2 (GELU)");
  if (ldx < K || ldy < N || (R && ldr < N)) return set_error(c, DI_EINVAL, "linear_lora: a row stride is shorter than its row");
  if (!aligned16(X) || !aligned16(W) || !aligned16(A) || !aligned16(B) || !aligned16(R) || !aligned16(Y) || ldx % 8 ||
      ldy % 8 || (R && ldr % 8))
    return set_error(c, DI_EINVAL, "linear_lora: pointers must be 16-byte aligned, row strides multiples of 8 elements");
  // blocks write Y while others still read X, or a residual that is not the same rows of Y
  if (rows_meet(X, ldx, K, Y, ldy, N, M) || (R && (R != Y || (M > 1 && ldr != ldy)) && rows_meet(R, ldr, N, Y, ldy, N, M)))
    return set_error(c, DI_EINVAL, "linear_lora: the output shares memory with x, or with a residual other than itself");
  if ((M + 127LL) / 128 * ((N + 31) / 32) > 0x7fffffffll)
    return set_error(c, DI_EUNSUPPORTED, "linear_lora: too many rows and columns");
  const size_t need = di_linear_lora_workspace(h, cfg);
  if (need && (!ws || ws_bytes < need || !aligned16(ws)))
    return set_error(c, DI_EINVAL, "linear_lora: workspace missing, too small or not 16-byte aligned");
  LoraParams p;
  memset(&p, 0, sizeof p);
  p.X = X; p.W = W; p.A = A; p.B = B; p.R = R; p.Y = Y;
  p.ldx = ldx; p.ldr = ldr; p.ldy = ldy;
  p.M = M; p.N = N; p.K = K; p.r = rank; p.L = L;
  p.scale = scale; p.bias = bias; p.rows = row_adapter; p.act = (int)act;
  p.err = c->d_err;
  p.T = static_cast<float*>(ws);
  p.T16 = static_cast<uint16_t*>(ws);
  if (M <= kSkinnyRows) return dtype == DI_F16 ? launch_skinny<false>(c, p) : launch_skinny<true>(c, p);
  return dtype == DI_F16 ? launch_tiles<false>(c, p) : launch_tiles<true>(c, p);
}
