// k_lora.cu — a linear layer with a low-rank adapter per row beside the shared weight (sm_100a).
//
//   Y[m] = act(X[m] W^T + bias + scale[a] (X[m] A[a]^T) B[a]^T) + R[m],   a = row_adapter[m]
//
// A negative index takes no adapter; an index past the last adapter takes none either and sets
// DEVERR_BOUNDS in the device error word.
//
// Tiles (M > kSkinnyRows): one persistent tensor-core kernel computes all of it in one pass over X.  A unit is a
// tile of 128 rows and BN columns.  The adapters that its rows name, each once, are its slots.  The B
// operand of the main loop is [W rows of the tile; A rows of the slots] in one shared-memory block, so one MMA
// of N = BN + slots * rank accumulates X W^T and X A^T together.  The second part, T, is then scaled,
// split into two 16-bit parts (hi + lo: 2^-17 relative for bf16) and written back to TMEM over itself, where it is
// the A operand of the products T B^T that add to the first part, each slot's in the lanes of its own rows only (so
// an adapter's infinities stay with its rows).  Those follow a few K blocks into the next unit's main loop,
// when T has been written, so the tensor pipe does not wait.
// More adapters in a tile than a pass has slots for take further passes over X with A rows alone.
//   warp 0       TMA loads through one ring of stages
//   warp 1       MMA issue
//   warp 2       slots of a unit: its distinct adapters and their rows, each row's scale
//   warps 4-7    T: TMEM -> scaled, 16-bit -> TMEM
//   warps 8-15   epilogue: bias, activation, residual, stores through shared memory by TMA
//
// Few rows (M <= kSkinnyRows): two launches.  The first computes T in 32 bits, the second streams W once from
// memory into mma.sync fragments (a tile of 16 weight rows by 8 rows of X), starting before the first is done, and adds
// the rows' own B products with plain FMAs: every byte of W, A and B is read about once, whoever owns it.
#include <algorithm>
#include <cstring>

#include "di_common.cuh"

namespace di {

struct LoraParams {
  CUtensorMap tmX, tmW, tmA, tmB, tmY;
  const void *X, *W, *A, *B, *R;
  void* Y;
  long long ldx, ldr, ldy;
  int M, N, K, r, L;
  const float *scale, *bias;
  const int* rows;
  int act;
  int* err;
  // tiles
  int BN, rp, slots, stages, mt, nt;  // rp: rank rounded up to 16; slots adapters per pass
  uint32_t stage_bytes;
  // few rows
  float* T;  // [M][r] scale[a] * X A^T
};

namespace {

constexpr int kSkinnyRows = 128;
constexpr int kLThreads = 512;
constexpr int kLists = 3;       // units whose slots are held
constexpr int kDefer = 4;       // K blocks of the next unit before this unit's T B^T products
constexpr int kMaxStages = 10;
constexpr uint32_t kSlab = 2048;  // 32 x 32 16-bit outputs of one epilogue warp

struct SlotList {
  int n;            // adapters in the unit
  int ids[128];
  uint4 others[128];  // per slot: the rows (TMEM lanes) that do not name its adapter
  float scale[128];   // per row
};
constexpr uint32_t kFixedSmem = 1024 + 8 * kSlab + ((kLists * sizeof(SlotList) + 15) / 16 * 16) + 512;

// D[tmem] += A[tmem] * B[smem desc] in all lanes but those of `off` (bit l of its words: lane l): A's 16-bit values lie
// two to a column, row m in lane m
__device__ __forceinline__ void umma_f16_ta_rows(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                                 const uint4& off) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.eq.b32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, "
      "{%4, %5, %6, %7}, p;\n\t}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(off.x), "r"(off.y), "r"(off.z), "r"(off.w)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
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
__device__ __forceinline__ float act_of(float v, int act) { return act == 1 ? silu_f(v) : act == 2 ? gelu_erf(v) : v; }

// Buffer index and phase of a ring.
struct Ring {
  int s = 0, ph = 0;
  __device__ __forceinline__ void advance(int n) {
    if (++s == n) { s = 0; ph ^= 1; }
  }
};

// Walks a CTA's stages in the order that the loader fills and the MMA warp drains them: K blocks of each pass, and
// the T B^T blocks of a pass at once, or, for a unit's last pass, kDefer K blocks into the next unit.
// kblock(pass, kb), pass_done(pass, count), expand(list slot, pass, count) return false to stop.
template <typename Begin, typename KBlock, typename PassDone, typename Expand, typename End>
__device__ __forceinline__ bool walk_units(const LoraParams& p, Begin begin, KBlock kblock, PassDone pass_done,
                                           Expand expand, End end) {
  const int units = p.mt * p.nt, nk = p.K / 64;
  int pend_pass = -1, pend_u = 0;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    int nd = 0;
    if (!begin(u, nd)) return false;
    const int passes = max(1, (nd + p.slots - 1) / p.slots);
    for (int ps = 0; ps < passes; ++ps) {
      const int cnt = min(p.slots, nd - ps * p.slots);
      for (int kb = 0; kb < nk; ++kb) {
        if (pend_pass >= 0 && kb == min(kDefer, nk - 1)) {
          if (!expand(pend_u, pend_pass)) return false;
          end(pend_u);
          pend_pass = -1;
        }
        if (!kblock(u, ps, kb, cnt)) return false;
      }
      pass_done(u, ps, cnt);
      if (cnt > 0) {
        if (ps == passes - 1) {
          pend_pass = ps;
          pend_u = u;
        } else if (!expand(u, ps)) {
          return false;
        }
      } else {
        end(u);
      }
    }
  }
  if (pend_pass >= 0) {
    if (!expand(pend_u, pend_pass)) return false;
    end(pend_u);
  }
  return true;
}

template <bool BF16>
__global__ void __launch_bounds__(kLThreads, 1) lora_tile_kernel(const __grid_constant__ LoraParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sStage = smem;                                    // [stages]: 128 X rows, then W and A rows, 128 B each
  uint8_t* sSlab = smem + p.stages * p.stage_bytes;          // [8]
  SlotList* lists = reinterpret_cast<SlotList*>(sSlab + 8 * kSlab);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sSlab + 8 * kSlab + (kLists * sizeof(SlotList) + 15) / 16 * 16);
  uint64_t* full = bars;                       // [kMaxStages]
  uint64_t* empty = full + kMaxStages;         // [kMaxStages]
  uint64_t* list_full = empty + kMaxStages;    // [kLists]
  uint64_t* list_empty = list_full + kLists;   // [kLists]
  uint64_t* t_ready = list_empty + kLists;     // [2] X A^T of accumulator ab complete
  uint64_t* t_full = t_ready + 2;              // [2] T written
  uint64_t* d_full = t_full + 2;               // [2] accumulator complete
  uint64_t* d_empty = d_full + 2;              // [2] accumulator read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < kLists; ++i) { mbar_init(&list_full[i], 1); mbar_init(&list_empty[i], 6); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&t_ready[i], 1);
      mbar_init(&t_full[i], 4);
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();
  const int units = p.mt * p.nt;
  // TMEM: accumulator ab of the unit's BN columns at 256 ab, its X A^T (then T) behind them

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tmX);
      tma_prefetch_desc(&p.tmW);
      tma_prefetch_desc(&p.tmA);
      tma_prefetch_desc(&p.tmB);
      Ring st, li, le;  // stages, lists begun, lists ended
      int cur = 0;      // list of the unit that is being loaded
      unsigned issued = 0;
      auto stage = [&]() {
        return !*abort_flag && mbar_wait(&empty[st.s], st.ph ^ 1, p.err, DEVERR_WAIT_TMA);
      };
      const bool ok = walk_units(
          p,
          [&](int u, int& nd) {
            if (*abort_flag || !mbar_wait(&list_full[li.s], li.ph, p.err, DEVERR_WAIT_TMA)) return false;
            cur = li.s;
            nd = lists[cur].n;
            li.advance(kLists);
            return true;
          },
          [&](int u, int ps, int kb, int cnt) {
            if (!stage()) return false;
            uint8_t* d = sStage + st.s * p.stage_bytes;
            mbar_arrive_expect_tx(&full[st.s], 16384u + (uint32_t)((ps == 0 ? p.BN : 0) + max(cnt, 0) * p.rp) * 128u);
            tma_load_2d(d, &p.tmX, &full[st.s], kb * 64, u / p.nt * 128);
            if (ps == 0) tma_load_2d(d + 16384, &p.tmW, &full[st.s], kb * 64, u % p.nt * p.BN);
            for (int g = 0; g < cnt; ++g)
              tma_load_3d(d + 16384 + (p.BN + g * p.rp) * 128, &p.tmA, &full[st.s], kb * 64, 0,
                          lists[cur].ids[ps * p.slots + g]);
            st.advance(p.stages);
            ++issued;
            return true;
          },
          [&](int, int, int) {},
          [&](int u, int ps) {
            const int cnt = min(p.slots, lists[le.s].n - ps * p.slots);
            for (int g = 0; g < cnt; ++g)
              for (int c = 0; c < p.rp; c += 64) {
                if (!stage()) return false;
                mbar_arrive_expect_tx(&full[st.s], (uint32_t)p.BN * 128u);
                tma_load_3d(sStage + st.s * p.stage_bytes + 16384, &p.tmB, &full[st.s], c, u % p.nt * p.BN,
                            lists[le.s].ids[ps * p.slots + g]);
                st.advance(p.stages);
                ++issued;
              }
            return true;
          },
          [&](int) {
            mbar_arrive(&list_empty[le.s]);
            le.advance(kLists);
          });
      if (!ok) {  // leave no copy in flight behind
        *abort_flag = 1;
        for (unsigned i = 0; i < min(issued, (unsigned)p.stages); ++i) {
          st.s = st.s ? st.s - 1 : (st.ph ^= 1, p.stages - 1);
          mbar_wait(&full[st.s], st.ph, p.err, DEVERR_WAIT_TMA);
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      Ring st, li, le;
      int ab_u = -1;          // accumulator of the unit in its main loop
      int nu = 0;             // units begun
      int eu = 0;             // units ended
      int ph_t[2] = {0, 0};
      auto stage = [&]() {
        return !*abort_flag && mbar_wait(&full[st.s], st.ph, p.err, DEVERR_WAIT_MMA);
      };
      const bool ok = walk_units(
          p,
          [&](int u, int& nd) {
            if (*abort_flag || !mbar_wait(&list_full[li.s], li.ph, p.err, DEVERR_WAIT_MMA)) return false;
            nd = lists[li.s].n;
            li.advance(kLists);
            ab_u = nu & 1;
            if (!mbar_wait(&d_empty[ab_u], ((nu >> 1) & 1) ^ 1, p.err, DEVERR_WAIT_MMA)) return false;
            ++nu;
            return true;
          },
          [&](int u, int ps, int kb, int cnt) {
            if (!stage()) return false;
            tc_fence_after();
            const uint32_t a = smem_u32(sStage + st.s * p.stage_bytes);
            const int first = ps == 0 ? 0 : p.BN, n = (ps == 0 ? p.BN : 0) + max(cnt, 0) * p.rp;
            const uint32_t id = idesc_f16(128, 0, BF16) | ((uint32_t)(n >> 3) << 17);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16(tmem + ab_u * 256 + first, sdesc_sw128(a + k * 32, 16, 1024),
                       sdesc_sw128(a + 16384 + first * 128 + k * 32, 16, 1024), id, (kb | k) != 0);
            umma_commit(&empty[st.s]);
            st.advance(p.stages);
            return true;
          },
          [&](int u, int ps, int cnt) { umma_commit(cnt > 0 ? &t_ready[ab_u] : &d_full[ab_u]); },
          [&](int u, int ps) {
            const int ab = eu & 1, nd = lists[le.s].n, cnt = min(p.slots, nd - ps * p.slots);
            if (*abort_flag || !mbar_wait(&t_full[ab], ph_t[ab], p.err, DEVERR_WAIT_MMA)) return false;
            ph_t[ab] ^= 1;
            const uint32_t d = tmem + ab * 256, t = d + p.BN;
            const uint32_t id = idesc_f16(128, 0, BF16) | ((uint32_t)(p.BN >> 3) << 17);
            for (int g = 0; g < cnt; ++g) {
              const uint4 off = lists[le.s].others[ps * p.slots + g];
              for (int c = 0; c < p.rp; c += 64) {
                if (!stage()) return false;
                tc_fence_after();
                const uint32_t b = smem_u32(sStage + st.s * p.stage_bytes + 16384);
                for (int k = 0; k < min(64, p.rp - c); k += 16) {
                  const int col = g * p.rp + c + k;  // 32 T columns: 16 of hi pairs, then 16 of lo pairs
                  const uint32_t at = t + col / 32 * 32 + col % 32 / 2;
                  const uint64_t bd = sdesc_sw128(b + k * 2, 16, 1024);
                  umma_f16_ta_rows(d, at, bd, id, off);
                  umma_f16_ta_rows(d, at + 16, bd, id, off);
                }
                umma_commit(&empty[st.s]);
                st.advance(p.stages);
              }
            }
            if ((ps + 1) * p.slots >= nd) umma_commit(&d_full[ab]);
            return true;
          },
          [&](int) {
            mbar_arrive(&list_empty[le.s]);
            le.advance(kLists);
            ++eu;
          });
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 2) {
    Ring li;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const bool ok = !*abort_flag && mbar_wait(&list_empty[li.s], li.ph ^ 1, p.err, DEVERR_WAIT_EPI);
      if (!__all_sync(0xffffffffu, ok)) { *abort_flag = 1; break; }
      SlotList& l = lists[li.s];
      int a[4];
      bool open_rows[4];  // rows whose adapter has no slot yet
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = u / p.nt * 128 + i * 32 + lane;
        a[i] = m < p.M ? __ldg(p.rows + m) : -1;
        if (a[i] >= p.L) {
          atomicOr(p.err, DEVERR_BOUNDS);
          a[i] = -1;
        }
        l.scale[i * 32 + lane] = a[i] >= 0 ? __ldg(p.scale + a[i]) : 0.f;
        open_rows[i] = a[i] >= 0;
      }
      int n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned open;
        while ((open = __ballot_sync(0xffffffffu, open_rows[i])) != 0) {
          const int id = __shfl_sync(0xffffffffu, a[i], __ffs(open) - 1);
          unsigned b[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            b[k] = __ballot_sync(0xffffffffu, a[k] != id);
            open_rows[k] = open_rows[k] && a[k] != id;
          }
          if (lane == 0) {
            l.ids[n] = id;
            l.others[n] = make_uint4(b[0], b[1], b[2], b[3]);
          }
          ++n;
        }
      }
      if (lane == 0) l.n = n;
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_full[li.s]);
      li.advance(kLists);
    }
  } else if (warp >= 4 && warp < 8) {
    const int q = warp & 3, row = q * 32 + lane;
    Ring li;
    int nu = 0, ph[2] = {0, 0};
    bool ok = true;
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x, ++nu) {
      ok = !*abort_flag && mbar_wait(&list_full[li.s], li.ph, p.err, DEVERR_WAIT_EPI);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int nd = lists[li.s].n, ab = nu & 1;
      const float sc = lists[li.s].scale[row];
      __syncwarp();
      if (lane == 0) mbar_arrive(&list_empty[li.s]);
      li.advance(kLists);
      const uint32_t t = tmem + ab * 256 + p.BN + (static_cast<uint32_t>(q * 32) << 16);
      for (int first = 0; first < nd; first += p.slots) {
        ok = !*abort_flag && mbar_wait(&t_ready[ab], ph[ab], p.err, DEVERR_WAIT_EPI);
        ok = __all_sync(0xffffffffu, ok);
        ph[ab] ^= 1;
        if (!ok) break;
        tc_fence_after();
        const int cols = min(p.slots, nd - first) * p.rp;
        for (int c = 0; c < cols; c += 32) {
          uint32_t r[32];
          tmem_ld32(t + c, r);
          tmem_wait_ld();
          uint32_t w[32];  // 16 hi pairs, 16 lo pairs
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const float x = sc * __uint_as_float(r[k]), y = sc * __uint_as_float(r[k + 1]);
            w[k / 2] = pack2<BF16>(x, y);
            const float2 h = unpack2<BF16>(w[k / 2]);
            // a part that is not finite stands alone (inf - inf would be NaN)
            w[16 + k / 2] = pack2<BF16>(isinf(h.x) ? 0.f : x - h.x, isinf(h.y) ? 0.f : y - h.y);
          }
          tmem_st32(t + c, w);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&t_full[ab]);
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp >= 8) {
    const int q = warp & 3, half = (warp - 8) / 4;
    uint8_t* slab = sSlab + (warp - 8) * kSlab;
    bool ok = true;
    int nu = 0;
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x, ++nu) {
      const int ab = nu & 1, m0 = u / p.nt * 128 + q * 32, n0 = u % p.nt * p.BN, m = m0 + lane;
      ok = !*abort_flag && mbar_wait(&d_full[ab], (nu >> 1) & 1, p.err, DEVERR_WAIT_EPI);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d = tmem + ab * 256 + (static_cast<uint32_t>(q * 32) << 16);
      if (m0 < p.M) {
#pragma unroll 1
        for (int c = half * 32; c < p.BN; c += 64) {
          const int nb = n0 + c;
          if (nb >= p.N) break;
          uint4 res[4];
          if (p.R && m < p.M) {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.R) + m * p.ldr + nb);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (nb + k * 8 < p.N) res[k] = src[k];  // may be the output: not through the read-only path
          }
          const float bl = p.bias && nb + lane < p.N ? __ldg(p.bias + nb + lane) : 0.f;
          uint32_t r[32];
          tmem_ld32(d + c, r);
          tmem_wait_ld();
          float v[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] = __uint_as_float(r[k]) + __shfl_sync(0xffffffffu, bl, k);
          if (p.act) {
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = act_of(v[k], p.act);
          }
          if (p.R && m < p.M) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t w[4] = {res[k].x, res[k].y, res[k].z, res[k].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<BF16>(w[e]);
                v[8 * k + 2 * e] += f.x;
                v[8 * k + 2 * e + 1] += f.y;
              }
            }
          }
          if (lane == 0) bulk_wait_read0();  // the previous chunk's store has read the slab
          __syncwarp();
          uint4* rp = reinterpret_cast<uint4*>(slab + lane * 64);  // 64-byte rows, 64-byte swizzle
#pragma unroll
          for (int k = 0; k < 4; ++k)
            rp[k ^ ((lane >> 1) & 3)] = make_uint4(pack2<BF16>(v[8 * k], v[8 * k + 1]), pack2<BF16>(v[8 * k + 2], v[8 * k + 3]),
                                                   pack2<BF16>(v[8 * k + 4], v[8 * k + 5]),
                                                   pack2<BF16>(v[8 * k + 6], v[8 * k + 7]));
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.tmY, slab, nb, m0);  // rows and columns outside Y are skipped
            bulk_commit();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&d_empty[ab]);
    }
    if (!ok) *abort_flag = 1;
    if (lane == 0) bulk_wait0();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- few rows ----

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
  const uint16_t* x = static_cast<const uint16_t*>(p.X) + m * p.ldx;
  const uint16_t* w = static_cast<const uint16_t*>(p.A) + ((long long)a * p.r + j) * p.K;
  float s = 0.f;
#pragma unroll 4
  for (int k = lane * 8; k < p.K; k += 256) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + k)), v = __ldg(reinterpret_cast<const uint4*>(w + k));
    const uint32_t uu[4] = {u.x, u.y, u.z, u.w}, vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2<BF16>(uu[e]), g = unpack2<BF16>(vv[e]);
      s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) p.T[m * p.r + j] = __ldg(p.scale + a) * s;
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

// 16 columns of Y for MT * 8 rows per block; the 8 warps take 32-wide K blocks in turn and are summed in shared memory.
// A lane's 16-byte loads of 8 consecutive k stand for two 16-wide MMA steps: both operands use the same order of k.
template <bool BF16, int MT>
__global__ void __launch_bounds__(256) lora_skinny_kernel(const __grid_constant__ LoraParams p) {
  __shared__ float red[8][MT * 8][17];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * MT * 8;
  // The shrink kernel lets this one start after its own wait for earlier kernels: X, W and B may be read at once,
  // T, R and Y only after it.
  pdl_trigger();
  float acc[MT][4] = {};
  const uint16_t* w0 = static_cast<const uint16_t*>(p.W) + (long long)(n0 + lane / 4) * p.K + (lane & 3) * 8;
  const uint16_t* w1 = w0 + 8ll * p.K;
  const uint16_t* x0 = static_cast<const uint16_t*>(p.X) + (lane & 3) * 8;
#pragma unroll 4
  for (int k = warp * 32; k < p.K; k += 256) {
    const uint4 a0 = __ldg(reinterpret_cast<const uint4*>(w0 + k)), a1 = __ldg(reinterpret_cast<const uint4*>(w1 + k));
    uint4 b[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = min(m0 + t * 8 + lane / 4, p.M - 1);  // rows past the last are computed and not stored
      b[t] = __ldg(reinterpret_cast<const uint4*>(x0 + m * p.ldx + k));
    }
    const uint32_t f0[4] = {a0.x, a1.x, a0.y, a1.y}, f1[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      mma_16x8x16<BF16>(acc[t], f0, b[t].x, b[t].y);
      mma_16x8x16<BF16>(acc[t], f1, b[t].z, b[t].w);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {  // d[0..1]: column lane / 4, rows 2 (lane & 3) + {0, 1}; d[2..3]: column + 8
    const int m = t * 8 + (lane & 3) * 2, n = lane / 4;
    red[warp][m][n] = acc[t][0];
    red[warp][m + 1][n] = acc[t][1];
    red[warp][m][n + 8] = acc[t][2];
    red[warp][m + 1][n + 8] = acc[t][3];
  }
  __syncthreads();
  pdl_wait();  // T is complete
  // outputs: groups of 2^g lanes share one output's rank chunks of 8
  int g = 0;
  while ((8 << g) < p.r) ++g;
  const int per = 256 >> g, sub = threadIdx.x & ((1 << g) - 1);
  for (int o = threadIdx.x >> g; o < (MT * 128 + per - 1) / per * per; o += per) {  // whole warps stay for the shuffles
    const int n = o & 15, ml = o >> 4, m = m0 + ml;
    const bool on = ml < MT * 8 && m < p.M;
    int a = on ? __ldg(p.rows + m) : -1;
    if (a >= p.L) a = -1;
    float s = 0.f;
    if (a >= 0 && sub * 8 < p.r) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.B) +
                                                           ((long long)a * p.N + n0 + n) * p.r + sub * 8));
      const float* t = p.T + m * p.r + sub * 8;
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<BF16>(w[e]);
        s = fmaf(t[2 * e], f.x, fmaf(t[2 * e + 1], f.y, s));
      }
    }
    for (int x = 1; x < (1 << g); x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    if (on && sub == 0) {
#pragma unroll
      for (int x = 0; x < 8; ++x) s += red[x][ml][n];
      if (p.bias) s += __ldg(p.bias + n0 + n);
      s = act_of(s, p.act);
      if (p.R) {
        const uint16_t v = static_cast<const uint16_t*>(p.R)[m * p.ldr + n0 + n];
        s += unpack2<BF16>(v).x;
      }
      static_cast<uint16_t*>(p.Y)[m * p.ldy + n0 + n] = (uint16_t)pack2<BF16>(s, 0.f);
    }
  }
}

template <bool BF16>
int launch_skinny(Ctx* c, const LoraParams& p) {
  launch_k(lora_shrink_kernel<BF16>, dim3(p.r / 8, p.M), 256, 0, c->stream, p);
  const int rc = check_launch(c, "linear_lora");
  if (rc != DI_OK) return rc;
  const int tiles = (p.M + 7) / 8;
  auto go = [&](auto kern, int mt) { launch_k(kern, dim3(p.N / 16, (tiles + mt - 1) / mt), 256, 0, c->stream, p); };
  if (tiles == 1) go(lora_skinny_kernel<BF16, 1>, 1);
  else if (tiles == 2) go(lora_skinny_kernel<BF16, 2>, 2);
  else if (tiles <= 4) go(lora_skinny_kernel<BF16, 4>, 4);
  else go(lora_skinny_kernel<BF16, 8>, 8);
  return check_launch(c, "linear_lora");
}

template <bool BF16>
int launch_tiles(Ctx* c, LoraParams& p) {
  p.rp = (p.r + 15) / 16 * 16;
  p.slots = std::max(1, std::min(64 / p.rp, p.L));
  p.mt = (p.M + 127) / 128;
  const int t_cols = (p.slots * p.rp + 31) / 32 * 32;
  // Column width: the K loop of a unit costs about its MMA columns or its stage's bytes over the shared-memory fill rate,
  // whichever is more, and a unit some 2500 cycles besides; the widest tile does not always fill the SMs.
  double best = 1e30;
  for (int bn = 32; bn <= 192 && bn + t_cols <= 256; bn += 32) {
    const int nt = (p.N + bn - 1) / bn;
    const double rounds = (double)(((long long)p.mt * nt + c->num_sms - 1) / c->num_sms);
    const double kb = std::max<double>(bn + p.rp, (16384 + (bn + p.rp) * 128) / 90.0);
    const double cost = rounds * (p.K / 64 * kb + 500.0) + 2000.0;
    if (cost < best * 0.999) {
      best = cost;
      p.BN = bn;
      p.nt = nt;
    }
  }
  p.stage_bytes = 16384 + (p.BN + p.slots * p.rp) * 128;
  p.stage_bytes = (p.stage_bytes + 1023) / 1024 * 1024;
  p.stages = (int)std::min<uint32_t>(kMaxStages, (232448 - kFixedSmem) / p.stage_bytes);
  const uint32_t smem = kFixedSmem + p.stages * p.stage_bytes;
  const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const uint64_t xd[2] = {(uint64_t)p.K, (uint64_t)p.M}, wd[2] = {(uint64_t)p.K, (uint64_t)p.N};
  const uint64_t ad[3] = {(uint64_t)p.K, (uint64_t)p.r, (uint64_t)p.L}, bd[3] = {(uint64_t)p.r, (uint64_t)p.N, (uint64_t)p.L};
  const uint64_t yd[2] = {(uint64_t)p.N, (uint64_t)p.M};
  const uint64_t xs[1] = {(uint64_t)p.ldx * 2}, wst[1] = {(uint64_t)p.K * 2}, ys[1] = {(uint64_t)p.ldy * 2};
  const uint64_t as[2] = {(uint64_t)p.K * 2, (uint64_t)p.r * p.K * 2}, bs[2] = {(uint64_t)p.r * 2, (uint64_t)p.N * p.r * 2};
  const uint32_t xb[2] = {64, 128}, wb[2] = {64, (uint32_t)p.BN}, ab[3] = {64, (uint32_t)p.rp, 1}, bb[3] = {64, (uint32_t)p.BN, 1},
                 yb[2] = {32, 32};
  std::string err;
  if (!make_tmap(&p.tmX, dt, 2, p.X, xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmW, dt, 2, p.W, wd, wst, wb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmA, dt, 3, p.A, ad, as, ab, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmB, dt, 3, p.B, bd, bs, bb, CU_TENSOR_MAP_SWIZZLE_128B, &err) ||
      !make_tmap(&p.tmY, dt, 2, p.Y, yd, ys, yb, CU_TENSOR_MAP_SWIZZLE_64B, &err))
    return set_error(c, DI_EINVAL, "linear_lora: " + err);
  auto kern = lora_tile_kernel<BF16>;
  static unsigned attr_done = 0;
  if (!(attr_done & (1u << (c->device & 31)))) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448) != cudaSuccess)
      return set_error(c, DI_ECUDA, "linear_lora: shared memory attribute");
    attr_done |= 1u << (c->device & 31);
  }
  launch_k(kern, dim3((unsigned)std::min<long long>((long long)p.mt * p.nt, c->num_sms)), kLThreads, smem, c->stream, p);
  return check_launch(c, "linear_lora");
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" size_t di_linear_lora_workspace(di_ctx_t h, int M, int N, int K, int rank, int n_adapters) {
  if (!h || M <= 0 || rank <= 0 || M > kSkinnyRows) return 0;
  return (size_t)M * rank * 4;
}

extern "C" int di_linear_lora(di_ctx_t h, int dtype, const void* X, long long ldx, int M, int K, const void* W, int N,
                              const void* A, const void* B, int rank, int n_adapters, const float* scale,
                              const int* row_adapter, const float* bias, const void* R, long long ldr, int act, void* Y,
                              long long ldy, void* ws, size_t ws_bytes) {
  Ctx* c = ctx_of(h);
  if (!c || (dtype != DI_F16 && dtype != DI_BF16)) return DI_EINVAL;
  DeviceGuard guard(c->device);
  if (M <= 0 || N <= 0 || K <= 0 || n_adapters <= 0 || !X || !W || !A || !B || !scale || !row_adapter || !Y)
    return set_error(c, DI_EINVAL, "linear_lora: bad shape or missing tensor");
  if (K % 64 || N % 16) return set_error(c, DI_EUNSUPPORTED, "linear_lora: K must be a multiple of 64, N of 16");
  if (rank < 8 || rank > 128 || rank % 8)
    return set_error(c, DI_EUNSUPPORTED, "linear_lora: the rank must be a multiple of 8, 8 to 128");
  if (act < 0 || act > 2) return set_error(c, DI_EINVAL, "linear_lora: act must be 0 (none), 1 (SiLU) or 2 (GELU)");
  if (ldx < K || ldy < N || (R && ldr < N)) return set_error(c, DI_EINVAL, "linear_lora: a row stride is shorter than its row");
  if (!aligned16(X) || !aligned16(W) || !aligned16(A) || !aligned16(B) || !aligned16(R) || !aligned16(Y) || ldx % 8 ||
      ldy % 8 || (R && ldr % 8))
    return set_error(c, DI_EINVAL, "linear_lora: pointers must be 16-byte aligned, row strides multiples of 8 elements");
  if ((long long)((M + 127LL) / 128) * ((N + 31) / 32) > 0x7fffffffll)
    return set_error(c, DI_EUNSUPPORTED, "linear_lora: too many rows and columns");
  const size_t need = di_linear_lora_workspace(h, M, N, K, rank, n_adapters);
  if (need && (!ws || ws_bytes < need || !aligned16(ws)))
    return set_error(c, DI_EINVAL, "linear_lora: workspace missing, too small or not 16-byte aligned");
  LoraParams p;
  memset(&p, 0, sizeof p);
  p.X = X; p.W = W; p.A = A; p.B = B; p.R = R; p.Y = Y;
  p.ldx = ldx; p.ldr = ldr; p.ldy = ldy;
  p.M = M; p.N = N; p.K = K; p.r = rank; p.L = n_adapters;
  p.scale = scale; p.bias = bias; p.rows = row_adapter; p.act = act;
  p.err = c->d_err;
  p.T = static_cast<float*>(ws);
  if (M <= kSkinnyRows) return dtype == DI_F16 ? launch_skinny<false>(c, p) : launch_skinny<true>(c, p);
  return dtype == DI_F16 ? launch_tiles<false>(c, p) : launch_tiles<true>(c, p);
}
