// k_xattn.cu — attention over an encoder's states, with lengths and a key mask per request (sm_100a).
//
//   O[b,i,h] = sum_j softmax_j(scale Q[b,i,h] . K[b,j,g]) V[b,j,g],  g = h / (H / Hkv),
//   over the valid keys j < min(kv_len[b], Skv) with key_mask[b][j] != 0
//
// A request without valid keys gives zero rows; query rows from q_len[b] on are not written.
#include <algorithm>
#include <cstring>

#include "di_common.cuh"

namespace di {

struct XattnParams {
  const void *Q, *K, *V;
  void* O;
  long long qs[3], ks[3], vs[3], os[3];  // batch, token, head strides in elements
  int B, H, G, Sq, Skv;
  const int *q_len, *kv_len;
  const unsigned char* mask;
  float scale_log2;
};

namespace {

template <typename E, int D>
__global__ void xattn_row_kernel(XattnParams p) {
  pdl_begin();
  const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (i >= (long long)p.B * p.H * p.Sq) return;
  const int s = (int)(i % p.Sq), h = (int)(i / p.Sq % p.H), b = (int)(i / p.Sq / p.H);
  if (p.q_len && s >= p.q_len[b]) return;
  const int n = p.kv_len ? min(p.kv_len[b], p.Skv) : p.Skv;
  constexpr int W = D / 32;
  float q[W], o[W] = {}, m = -INFINITY, l = 0.f;
  const E* qp = static_cast<const E*>(p.Q) + b * p.qs[0] + s * p.qs[1] + h * p.qs[2];
  for (int e = 0; e < W; ++e) q[e] = to_f(qp[lane + 32 * e]) * p.scale_log2;
  const E* kp = static_cast<const E*>(p.K) + b * p.ks[0] + (h / p.G) * p.ks[2];
  const E* vp = static_cast<const E*>(p.V) + b * p.vs[0] + (h / p.G) * p.vs[2];
  for (int j = 0; j < n; ++j) {
    if (p.mask && !p.mask[(long long)b * p.Skv + j]) continue;
    float d = 0.f;
    for (int e = 0; e < W; ++e) d = fmaf(q[e], to_f(kp[j * p.ks[1] + lane + 32 * e]), d);
    for (int w = 16; w; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
    const float mn = fmaxf(m, d), a = m == mn ? 1.f : exp2f(m - mn), x = exp2f(d - mn);
    l = l * a + x;
    for (int e = 0; e < W; ++e) o[e] = o[e] * a + x * to_f(vp[j * p.vs[1] + lane + 32 * e]);
    m = mn;
  }
  E* op = static_cast<E*>(p.O) + b * p.os[0] + s * p.os[1] + h * p.os[2];
  for (int e = 0; e < W; ++e) op[lane + 32 * e] = from_f<E>(l == 0.f ? 0.f : o[e] / l);
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" size_t di_cross_attention_workspace(di_ctx_t h, int B, int H, int Hkv, int Sq, int Skv, int D) {
  return 0;
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
  XattnParams p;
  memset(&p, 0, sizeof p);
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(O))
    return set_error(c, DI_EINVAL, "cross_attention: pointers must be 16-byte aligned");
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i]; p.ks[i] = k_strides[i]; p.vs[i] = v_strides[i]; p.os[i] = o_strides[i];
    if (p.qs[i] < 0 || p.ks[i] < 0 || p.vs[i] < 0 || p.os[i] < 0 || (p.qs[i] | p.ks[i] | p.vs[i] | p.os[i]) % 8)
      return set_error(c, DI_EINVAL, "cross_attention: strides must be multiples of 8 elements and not negative");
  }
  if (!(scale > 0.f) || !(scale < INFINITY)) return set_error(c, DI_EINVAL, "cross_attention: scale must be positive and finite");
  if ((p.os[0] == 0 && B > 1) || (p.os[1] == 0 && Sq > 1) || (p.os[2] == 0 && H > 1))
    return set_error(c, DI_EINVAL, "cross_attention: the output's rows must not share memory");
  p.Q = Q; p.K = K; p.V = V; p.O = O;
  p.B = B; p.H = H; p.G = H / Hkv; p.Sq = Sq; p.Skv = Skv;
  p.q_len = q_len; p.kv_len = kv_len; p.mask = key_mask;
  p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid((unsigned)(((long long)B * H * Sq * 32 + 255) / 256));
  if (dtype == DI_F16) {
    if (D == 64) launch_k(xattn_row_kernel<__half, 64>, grid, 256, 0, c->stream, p);
    else launch_k(xattn_row_kernel<__half, 128>, grid, 256, 0, c->stream, p);
  } else {
    if (D == 64) launch_k(xattn_row_kernel<__nv_bfloat16, 64>, grid, 256, 0, c->stream, p);
    else launch_k(xattn_row_kernel<__nv_bfloat16, 128>, grid, 256, 0, c->stream, p);
  }
  return check_launch(c, "cross_attention");
}
