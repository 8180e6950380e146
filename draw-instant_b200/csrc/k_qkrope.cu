// k_qkrope.cu — RMS norm of query and key heads with the rotation by position axes in the same pass (sm_100a).
//
//   y = rotate(x * rsqrt(mean(x^2) + eps) * w, pos)   per token and head, x of D = 64 or 128 values
//
// Pair i of a head (D/2 pairs) belongs to one position axis: the axes take d_0/2, d_1/2, ... pairs in turn
// (sum d_a = D) and pair j of axis a turns by pos[token][a] * theta^(-2j / d_a) radians.  A pair is two
// neighbouring values (interleaved) or values i and i + D/2 (halves).
//
// Bound: HBM, every value read and written once; at 23 bytes a cycle and SM that leaves some 170 instructions for the
// 1 KB that a warp reads and writes per step, so the arithmetic is packed (two values per instruction) and the
// angles are taken once per token for all its heads.  A warp takes four tokens (two at D = 128) side by side and walks their
// heads, queries then keys: a lane owns the same 8-value chunk of every head of one token, with the weights times the
// sines and cosines of its pairs in registers, and all traffic is whole 128-byte lines.  Loads run four steps ahead, and
// two steps go side by side: their shuffles and roots hide one another (65536 tokens of 5 + 5 heads of 64, fp16: 33.8 us,
// 5.0 TB/s; one at a time 38.7.  21600 tokens of 16 + 4 heads of 128, bf16: 41.5 us, 5.3 TB/s; 45.8).  Rotated halves
// exchange all values by shuffles (eight per 16 bytes) and run five blocks per SM instead of six: 40.0 and 45.4 us.
// The angle is the product of an integer position and a 64-bit frequency in turns, reduced to half a turn in 64 bits
// before the 32-bit sine (absolute error 2^-20.9): positions of any size keep the accuracy of position zero.
// Sums and products are 32-bit; the result is rounded once.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "di_common.cuh"

namespace di {

namespace {

constexpr int kMaxPairs = 64;  // D / 2 of the larger head

struct QkParams {
  const void* x[2];       // queries, keys
  void* y[2];
  long long ldx[2], ldy[2];  // token strides in elements; the heads of a token are contiguous
  const float* w[2];      // norm weights [D], or null: no norm
  int H[2];
  long long T;            // tokens
  int P, axes;            // rows and columns of pos
  const int* pos;         // null: no rotation
  float eps;
  int hsplit;             // warps that share a token's heads
  double freq[kMaxPairs];           // turns per position step
  unsigned char axis[kMaxPairs];
};

constexpr int kQkWarps = 4, kQkAhead = 4;  // warps per block, steps in flight

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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<__half2*>(&w));
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (std::is_same<T, __half>::value) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T, int D, bool HALVES>
__global__ void __launch_bounds__(32 * kQkWarps, HALVES ? 5 : 6) qk_norm_rope_kernel(const __grid_constant__ QkParams p) {
  constexpr int LPH = D / 8;   // lanes per head
  constexpr int TPW = 32 / LPH;  // tokens per warp
  const int lane = threadIdx.x & 31, chunk = lane % LPH;
  const int heads = p.H[0] + p.H[1];
  unsigned group = blockIdx.x * kQkWarps + (threadIdx.x >> 5);
  int h0 = 0, h1 = heads;
  if (p.hsplit > 1) {  // divisions are dear next to a warp's work: 32 bits, and only where they are needed
    const unsigned part = group % p.hsplit;
    group /= p.hsplit;
    h0 = (int)((unsigned)heads * part / p.hsplit);
    h1 = (int)((unsigned)heads * (part + 1) / p.hsplit);
  }
  const long long t = (long long)group * TPW + lane / LPH;
  const bool on = t < p.T;
  // A lane's 8 values are 4 pairs (interleaved), or one value each of 8 pairs whose other values lie LPH / 2 lanes on
  // (halves); it takes the angles of 4 pairs, in the halves' case 4 of the 8 and the other lane the rest.
  const int pair0 = HALVES ? chunk % (LPH / 2) * 8 + chunk / (LPH / 2) * 4 : chunk * 4;
  pdl_begin();
  // This warp's query heads and key heads, the queries padded to whole pairs of steps: step v of the two lists laid end to
  // end uses buffer v % kQkAhead.
  const int q0 = min(h0, p.H[0]), nq = min(h1, p.H[0]) - q0, k0 = max(h0 - p.H[0], 0), nk = max(h1 - p.H[0], 0) - k0;
  const int qpad = (nq + 1) / 2 * 2, steps = qpad + nk;
  const long long tt = on ? t : 0;
  const T* xq = static_cast<const T*>(p.x[0]) + tt * p.ldx[0] + (long long)q0 * D + chunk * 8;
  const T* xk = static_cast<const T*>(p.x[1]) + tt * p.ldx[1] + (long long)(k0 - qpad) * D + chunk * 8;
  T* y = nullptr;  // step v of the list at hand at y + v D
  uint4 raw[kQkAhead];
  auto fetch = [&](uint4& r, int v) {
    if (on && (v < nq || (v >= qpad && v < steps))) r = *reinterpret_cast<const uint4*>((v < qpad ? xq : xk) + (long long)v * D);
  };
#pragma unroll
  for (int u = 0; u < kQkAhead; ++u) fetch(raw[u], u);
  float co[HALVES ? 8 : 4], si[HALVES ? 8 : 4];
  if (p.pos) {
    const int* row = p.pos + (long long)(on ? (unsigned)t % (unsigned)p.P : 0u) * p.axes;
    float c4[4], s4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double turns = (double)__ldg(row + p.axis[pair0 + i]) * p.freq[pair0 + i];
      __sincosf(6.283185307f * (float)(turns - rint(turns)), &s4[i], &c4[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (HALVES) {
        const float oc = __shfl_xor_sync(0xffffffffu, c4[i], LPH / 2), os = __shfl_xor_sync(0xffffffffu, s4[i], LPH / 2);
        const bool low = chunk < LPH / 2;
        co[i % (HALVES ? 8 : 4)] = low ? c4[i] : oc;
        si[i % (HALVES ? 8 : 4)] = low ? s4[i] : os;
        co[(i + 4) % (HALVES ? 8 : 4)] = low ? oc : c4[i];
        si[(i + 4) % (HALVES ? 8 : 4)] = low ? os : s4[i];
      } else {
        co[i] = c4[i];
        si[i] = s4[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < (HALVES ? 8 : 4); ++i) { co[i] = 1.f; si[i] = 0.f; }
  }
  // Values two and two: interleaved, the first and the second values of pairs 2 j and 2 j + 1; halves, values 2 j and 2 j + 1.
  // With the weights folded in: first' = first * m1 + second * m2, second' = first * m3 + second * m4 (halves: own value
  // and other value times m1 and m2).
  uint64_t m1[HALVES ? 4 : 2], m2[HALVES ? 4 : 2], m3[2], m4[2];
  bool norm = false;
  auto list = [&](int l) {  // on to the queries, or the keys
    y = static_cast<T*>(p.y[l]) + (on ? t : 0) * p.ldy[l] + (long long)(l ? k0 - qpad : q0) * D + chunk * 8;
    const float* wp = p.w[l];
    norm = wp != nullptr;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = wp ? __ldg(wp + chunk * 8 + e) : 1.f;
#pragma unroll
    for (int j = 0; j < (HALVES ? 4 : 2); ++j) {
      if (HALVES) {
        const float sign = chunk < LPH / 2 ? -1.f : 1.f;
        const float o0 = __shfl_xor_sync(0xffffffffu, w[2 * j], LPH / 2), o1 = __shfl_xor_sync(0xffffffffu, w[2 * j + 1], LPH / 2);
        m1[j] = f2_pack(w[2 * j] * co[2 * j], w[2 * j + 1] * co[2 * j + 1]);
        m2[j] = f2_pack(sign * o0 * si[2 * j], sign * o1 * si[2 * j + 1]);
      } else {
        const float c0 = co[2 * j], c1 = co[2 * j + 1], s0 = si[2 * j], s1 = si[2 * j + 1];
        m1[j] = f2_pack(w[4 * j] * c0, w[4 * j + 2] * c1);
        m2[j] = f2_pack(-w[4 * j + 1] * s0, -w[4 * j + 3] * s1);
        m3[j] = f2_pack(w[4 * j] * s0, w[4 * j + 2] * s1);
        m4[j] = f2_pack(w[4 * j + 1] * c0, w[4 * j + 3] * c1);
      }
    }
  };
  // N steps side by side: their chains of shuffles hide one another.
  auto work = [&](auto count, uint4* r, int v) {
    constexpr int N = decltype(count)::value;
    uint64_t x[N][4], r2[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t w[4] = {r[n].x, r[n].y, r[n].z, r[n].w};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 f = unpack2<T>(w[2 * j]), g = unpack2<T>(w[2 * j + 1]);
        x[n][2 * j] = HALVES ? f2_pack(f.x, f.y) : f2_pack(f.x, g.x);
        x[n][2 * j + 1] = HALVES ? f2_pack(g.x, g.y) : f2_pack(f.y, g.y);
      }
    }
    fetch(r[0], v + kQkAhead);
    fetch(r[1], v + kQkAhead + 1);
    if (norm) {
      float ss[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const uint64_t q = fma2(x[n][0], x[n][0], fma2(x[n][1], x[n][1], fma2(x[n][2], x[n][2], mul2(x[n][3], x[n][3]))));
        ss[n] = lo_f(q) + hi_f(q);
      }
#pragma unroll
      for (int o = LPH / 2; o; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) ss[n] += __shfl_xor_sync(0xffffffffu, ss[n], o);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float s = rsqrtf(fmaf(ss[n], 1.0f / D, p.eps));
        r2[n] = f2_pack(s, s);
      }
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) r2[n] = f2_pack(1.f, 1.f);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t out[4];
      if (HALVES) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint64_t z = mul2(x[n][j], m1[j]);
          if (p.pos) {
            const uint64_t o = f2_pack(__shfl_xor_sync(0xffffffffu, lo_f(x[n][j]), LPH / 2),
                                       __shfl_xor_sync(0xffffffffu, hi_f(x[n][j]), LPH / 2));
            z = fma2(o, m2[j], z);
          }
          z = mul2(z, r2[n]);
          out[j] = pack2<T>(lo_f(z), hi_f(z));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint64_t f = x[n][2 * j], g = x[n][2 * j + 1];
          uint64_t f1 = mul2(f, m1[j]), g1 = mul2(g, m4[j]);
          if (p.pos) {
            f1 = fma2(g, m2[j], f1);
            g1 = fma2(f, m3[j], g1);
          }
          f1 = mul2(f1, r2[n]);
          g1 = mul2(g1, r2[n]);
          out[2 * j] = pack2<T>(lo_f(f1), lo_f(g1));
          out[2 * j + 1] = pack2<T>(hi_f(f1), hi_f(g1));
        }
      }
      if (on) *reinterpret_cast<uint4*>(y + (long long)(v + n) * D) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  };
#pragma unroll 1
  for (int v0 = 0; v0 < steps; v0 += kQkAhead)
#pragma unroll
    for (int u = 0; u < kQkAhead; u += 2) {
      const int v = v0 + u, left = (v < qpad ? nq : steps) - v;
      if (left <= 0) break;  // past the keys
      if (v == 0 || v == qpad) list(v >= qpad);
      if (left >= 2) work(std::integral_constant<int, 2>(), raw + u, v);
      else work(std::integral_constant<int, 1>(), raw + u, v);
    }
}

template <typename T, int D>
int launch_qk(Ctx* c, QkParams& p, int halves) {
  constexpr int TPW = 256 / D;
  // Few tokens: their heads are shared out over warps until the card has some 8 warps per SM.
  const long long groups = (p.T + TPW - 1) / TPW;
  p.hsplit = (int)std::max<long long>(1, std::min<long long>(p.H[0] + p.H[1], 8LL * c->num_sms / groups));
  const long long blocks = (groups * p.hsplit + kQkWarps - 1) / kQkWarps;
  auto kern = halves ? qk_norm_rope_kernel<T, D, true> : qk_norm_rope_kernel<T, D, false>;
  launch_k(kern, dim3((unsigned)blocks), dim3(32 * kQkWarps), 0, c->stream, p);
  return check_launch(c, "qk_norm_rope");
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" int di_qk_norm_rope(di_ctx_t h, int dtype, const long long cfg[14], float eps, double theta, const void* Q,
                               const void* K, const float* q_weight, const float* k_weight, const int* positions, void* Qo,
                               void* Ko) {
  Ctx* c = ctx_of(h);
  if (!c || (dtype != DI_F16 && dtype != DI_BF16)) return DI_EINVAL;
  DeviceGuard guard(c->device);
  if (!cfg || cfg[0] <= 0 || cfg[0] > 0x7fffffff || cfg[1] <= 0 || cfg[1] > 16384 || cfg[2] < 0 || cfg[2] > 16384 || !Q || !Qo ||
      (cfg[2] > 0) != (K != nullptr) || (cfg[2] > 0) != (Ko != nullptr))
    return set_error(c, DI_EINVAL, "qk_norm_rope: bad shape or missing tensor");
  const int T = (int)cfg[0], Hq = (int)cfg[1], Hk = (int)cfg[2];
  const long long D = cfg[3], ldq = cfg[4], ldk = cfg[5], ldqo = cfg[6], ldko = cfg[7];
  const long long pos_rows = cfg[8], pairing = cfg[9], n_axes = cfg[10], *axis_dims = cfg + 11;
  if (D != 64 && D != 128) return set_error(c, DI_EUNSUPPORTED, "qk_norm_rope: head dim must be 64 or 128");
  if (ldq < (long long)Hq * D || ldqo < (long long)Hq * D || (Hk && (ldk < (long long)Hk * D || ldko < (long long)Hk * D)))
    return set_error(c, DI_EINVAL, "qk_norm_rope: a token stride is shorter than the token's heads");
  if (!aligned16(Q) || !aligned16(Qo) || !aligned16(K) || !aligned16(Ko) || ldq % 8 || ldqo % 8 ||
      (Hk && (ldk % 8 || ldko % 8)))
    return set_error(c, DI_EINVAL, "qk_norm_rope: pointers must be 16-byte aligned, strides multiples of 8 elements");
  // a head is written where it was read, or elsewhere: never over another that is still to be read
  auto over = [T, D](const void* x, long long ldx, int hx, const void* y, long long ldy, int hy, bool itself) {
    return hx && hy && !(itself && x == y && (T == 1 || ldx == ldy)) && rows_meet(x, ldx, hx * D, y, ldy, hy * D, T);
  };
  if (over(Q, ldq, Hq, Qo, ldqo, Hq, true) || over(K, ldk, Hk, Ko, ldko, Hk, true) || over(Q, ldq, Hq, Ko, ldko, Hk, false) ||
      over(K, ldk, Hk, Qo, ldqo, Hq, false) || over(Qo, ldqo, Hq, Ko, ldko, Hk, false))
    return set_error(c, DI_EINVAL, "qk_norm_rope: an output shares memory with the other one, or with an input that is not its own");
  if (pairing != 0 && pairing != 1) return set_error(c, DI_EINVAL, "qk_norm_rope: pairing must be 0 or 1");
  if (!(eps >= 0.f)) return set_error(c, DI_EINVAL, "qk_norm_rope: eps must not be negative");
  QkParams p;
  memset(&p, 0, sizeof p);
  if (positions) {
    if (n_axes < 1 || n_axes > 3 || pos_rows < 1 || pos_rows > 0x7fffffff || !(theta > 0.0))
      return set_error(c, DI_EINVAL, "qk_norm_rope: needs 1 to 3 axes, their dims, position rows and theta > 0");
    int i = 0, sum = 0;
    for (int a = 0; a < n_axes; ++a) {
      if (axis_dims[a] < 2 || axis_dims[a] % 2 || axis_dims[a] > D - sum)
        return set_error(c, DI_EINVAL, "qk_norm_rope: axis dims must be even, positive and sum to the head dim");
      sum += (int)axis_dims[a];
      const long double ratio = std::pow((long double)theta, -2.0L / axis_dims[a]);
      long double f = 0.159154943091895335768883763372514362L;  // 1 / (2 pi); 64-bit products stay exact to 53 bits
      for (int j = 0; j < axis_dims[a] / 2; ++j, ++i, f *= ratio) {
        p.freq[i] = (double)f;
        p.axis[i] = (unsigned char)a;
      }
    }
    if (sum != D) return set_error(c, DI_EINVAL, "qk_norm_rope: axis dims must be even, positive and sum to the head dim");
  }
  p.x[0] = Q; p.x[1] = K;
  p.y[0] = Qo; p.y[1] = Ko;
  p.ldx[0] = ldq; p.ldx[1] = ldk;
  p.ldy[0] = ldqo; p.ldy[1] = ldko;
  p.w[0] = q_weight; p.w[1] = k_weight;
  p.H[0] = Hq; p.H[1] = Hk;
  p.T = T;
  p.P = positions ? (int)pos_rows : 1;
  p.axes = (int)n_axes;
  p.pos = positions;
  p.eps = eps;
  if (dtype == DI_F16) return D == 64 ? launch_qk<__half, 64>(c, p, (int)pairing) : launch_qk<__half, 128>(c, p, (int)pairing);
  return D == 64 ? launch_qk<__nv_bfloat16, 64>(c, p, (int)pairing) : launch_qk<__nv_bfloat16, 128>(c, p, (int)pairing);
}
