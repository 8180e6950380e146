// k_qkrope.cu — RMS norm of query and key heads with the rotation by position axes in the same pass (sm_100a).
//
//   y = rotate(x * rsqrt(mean(x^2) + eps) * w, pos)   per token and head, x of D = 64 or 128 values
//
// Pair i of a head (D/2 pairs) belongs to one position axis: the axes take d_0/2, d_1/2, ... pairs in turn
// (sum d_a = D) and pair j of axis a turns by pos[token][a] * theta^(-2j / d_a) radians.  A pair is two
// neighbouring values (interleaved) or values i and i + D/2 (halves).
//
// Bound: HBM, every value read and written once.  One warp takes one token at a time: a lane owns the same
// 8-value chunk of every head it meets, so the token's angles (one sine and cosine per pair, taken once per
// token for all its heads) and the weights stay in its registers, and all traffic is 16-byte accesses.
// The angle is the product of an integer position and a 64-bit frequency in turns, reduced to half a turn in 64
// bits before the 32-bit sine: positions of any size keep the accuracy of position zero.
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
  int tokens;             // tokens per warp
  double freq[kMaxPairs];           // turns per position step
  unsigned char axis[kMaxPairs];
};

constexpr int kQkWarps = 4, kQkTokens = 4, kQkUnroll = 4;  // warps per block, most tokens per warp, chunks in flight

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v = w[i];
    float2 t;
    if (std::is_same<T, __half>::value) t = __half22float2(*reinterpret_cast<__half2*>(&v));
    else t = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<T, __half>::value) {
      __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    } else {
      __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int D, bool HALVES>
__global__ void __launch_bounds__(32 * kQkWarps) qk_norm_rope_kernel(const __grid_constant__ QkParams p) {
  constexpr int LPH = D / 8;        // lanes per head
  constexpr int HPW = 32 / LPH;     // heads per warp step
  constexpr int PPL = D / 64;       // pairs whose angle a lane computes
  constexpr int NP = HALVES ? 8 : 4;  // pairs that a lane's chunk meets
  const int lane = threadIdx.x & 31;
  const long long warp = (long long)blockIdx.x * kQkWarps + (threadIdx.x >> 5);
  const int part = (int)(warp % p.hsplit);
  const long long t0 = warp / p.hsplit * p.tokens;
  const int chunk = lane % LPH, sub = lane / LPH;
  double fr[PPL];
  int ax[PPL];
#pragma unroll
  for (int i = 0; i < PPL; ++i) {
    fr[i] = p.freq[lane + 32 * i];
    ax[i] = p.axis[lane + 32 * i];
  }
  pdl_begin();
  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = p.w[0] ? __ldg(p.w[0] + chunk * 8 + e) : 1.f;
    wk[e] = p.w[1] ? __ldg(p.w[1] + chunk * 8 + e) : 1.f;
  }
  const int heads = p.H[0] + p.H[1], steps = (heads + HPW - 1) / HPW;
  const int s0 = (int)((long long)steps * part / p.hsplit), s1 = (int)((long long)steps * (part + 1) / p.hsplit);
  for (long long t = t0; t < min(t0 + p.tokens, p.T); ++t) {
    float c[NP], s[NP];
    if (p.pos) {
      float cl[PPL], sl[PPL];
#pragma unroll
      for (int i = 0; i < PPL; ++i) {
        const double turns = (double)__ldg(p.pos + (t % p.P) * p.axes + ax[i]) * fr[i];
        sincospif(2.0f * (float)(turns - rint(turns)), &sl[i], &cl[i]);
      }
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        // pair of this chunk's e-th value (halves) or value pair (interleaved), held by lane pair % 32
        const int pair = HALVES ? (chunk * 8 + e) % (D / 2) : chunk * 4 + e;
        c[e] = __shfl_sync(0xffffffffu, cl[0], pair & 31);
        s[e] = __shfl_sync(0xffffffffu, sl[0], pair & 31);
        if (PPL == 2) {
          const float c1 = __shfl_sync(0xffffffffu, cl[PPL - 1], pair & 31);
          const float s1v = __shfl_sync(0xffffffffu, sl[PPL - 1], pair & 31);
          if (pair >= 32) { c[e] = c1; s[e] = s1v; }
        }
      }
    }
    for (int st = s0; st < s1; st += kQkUnroll) {
      uint4 raw[kQkUnroll];
#pragma unroll
      for (int u = 0; u < kQkUnroll; ++u) {
        const int h = (st + u) * HPW + sub;
        raw[u] = make_uint4(0, 0, 0, 0);
        if (st + u < s1 && h < heads) {
          const int k = h >= p.H[0];
          raw[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x[k]) + t * p.ldx[k] +
                                                   (long long)(k ? h - p.H[0] : h) * D + chunk * 8);
        }
      }
#pragma unroll
      for (int u = 0; u < kQkUnroll; ++u) {
        if (st + u >= s1) break;  // warp-uniform
        const int h = (st + u) * HPW + sub;
        const int k = h >= p.H[0];
        float f[8];
        unpack8<T>(raw[u], f);
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
        for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (p.w[k]) {
          const float r = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= r * (k ? wk[e] : wq[e]);
        }
        if (p.pos) {
          if (HALVES) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float o = __shfl_xor_sync(0xffffffffu, f[e], LPH / 2);  // the pair's other value
              f[e] = chunk < LPH / 2 ? f[e] * c[e] - o * s[e] : o * s[e] + f[e] * c[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float lo = f[2 * e], hi = f[2 * e + 1];
              f[2 * e] = lo * c[e] - hi * s[e];
              f[2 * e + 1] = lo * s[e] + hi * c[e];
            }
          }
        }
        if (h < heads)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.y[k]) + t * p.ldy[k] + (long long)(k ? h - p.H[0] : h) * D +
                                    chunk * 8) = pack8<T>(f);
      }
    }
  }
}

template <typename T, int D>
int launch_qk(Ctx* c, const QkParams& p, int halves) {
  const long long groups = (p.T + p.tokens - 1) / p.tokens;
  const long long blocks = (groups * p.hsplit + kQkWarps - 1) / kQkWarps;
  auto kern = halves ? qk_norm_rope_kernel<T, D, true> : qk_norm_rope_kernel<T, D, false>;
  launch_k(kern, dim3((unsigned)blocks), dim3(32 * kQkWarps), 0, c->stream, p);
  return check_launch(c, "qk_norm_rope");
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" int di_qk_norm_rope(di_ctx_t h, int dtype, const void* Q, long long ldq, int Hq, const void* K,
                               long long ldk, int Hk, int T, int D, const float* q_weight, const float* k_weight,
                               float eps, const int* positions, int pos_rows, int n_axes, const int* axis_dims,
                               double theta, int pairing, void* Qo, long long ldqo, void* Ko, long long ldko) {
  Ctx* c = ctx_of(h);
  if (!c || (dtype != DI_F16 && dtype != DI_BF16)) return DI_EINVAL;
  DeviceGuard guard(c->device);
  if (T <= 0 || Hq <= 0 || Hk < 0 || !Q || !Qo || (Hk > 0) != (K != nullptr) || (Hk > 0) != (Ko != nullptr))
    return set_error(c, DI_EINVAL, "qk_norm_rope: bad shape or missing tensor");
  if (D != 64 && D != 128) return set_error(c, DI_EUNSUPPORTED, "qk_norm_rope: head dim must be 64 or 128");
  if (Hq + (long long)Hk > 65536) return set_error(c, DI_EINVAL, "qk_norm_rope: more than 65536 heads");
  if (ldq < (long long)Hq * D || ldqo < (long long)Hq * D || (Hk && (ldk < (long long)Hk * D || ldko < (long long)Hk * D)))
    return set_error(c, DI_EINVAL, "qk_norm_rope: a token stride is shorter than the token's heads");
  if (!aligned16(Q) || !aligned16(Qo) || !aligned16(K) || !aligned16(Ko) || ldq % 8 || ldqo % 8 ||
      (Hk && (ldk % 8 || ldko % 8)))
    return set_error(c, DI_EINVAL, "qk_norm_rope: pointers must be 16-byte aligned, strides multiples of 8 elements");
  if (pairing != 0 && pairing != 1) return set_error(c, DI_EINVAL, "qk_norm_rope: pairing must be 0 or 1");
  if (!(eps >= 0.f)) return set_error(c, DI_EINVAL, "qk_norm_rope: eps must not be negative");
  QkParams p;
  memset(&p, 0, sizeof p);
  if (positions) {
    if (n_axes < 1 || n_axes > 3 || pos_rows < 1 || !axis_dims || !(theta > 0.0))
      return set_error(c, DI_EINVAL, "qk_norm_rope: needs 1 to 3 axes, their dims, position rows and theta > 0");
    int i = 0, sum = 0;
    for (int a = 0; a < n_axes; ++a) {
      if (axis_dims[a] < 2 || axis_dims[a] % 2 || axis_dims[a] > D - sum)
        return set_error(c, DI_EINVAL, "qk_norm_rope: axis dims must be even, positive and sum to the head dim");
      sum += axis_dims[a];
      for (int j = 0; j < axis_dims[a] / 2; ++j, ++i) {
        p.freq[i] = std::pow(theta, -2.0 * j / axis_dims[a]) * 0.15915494309189533577;  // 1 / (2 pi)
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
  p.P = positions ? pos_rows : 1;
  p.axes = n_axes;
  p.pos = positions;
  p.eps = eps;
  // A warp keeps its pairs' frequencies over a few tokens when there are enough of them for 32 warps per SM;
  // few tokens share out their heads over warps until the card has some 8 warps per SM.
  p.tokens = (int)std::max<long long>(1, std::min<long long>(kQkTokens, T / (32LL * c->num_sms)));
  const int steps = (Hq + Hk + 256 / D - 1) / (256 / D);
  const long long groups = ((long long)T + p.tokens - 1) / p.tokens;
  p.hsplit = (int)std::max<long long>(1, std::min<long long>(steps, 8LL * c->num_sms / groups));
  if (dtype == DI_F16) return D == 64 ? launch_qk<__half, 64>(c, p, pairing) : launch_qk<__half, 128>(c, p, pairing);
  return D == 64 ? launch_qk<__nv_bfloat16, 64>(c, p, pairing) : launch_qk<__nv_bfloat16, 128>(c, p, pairing);
}
