// k_lora.cu — a linear layer with a low-rank adapter per row beside the shared weight (sm_100a).
//
//   Y[m] = act(X[m] W^T + bias + scale[a] (X[m] A[a]^T) B[a]^T) + R[m],   a = row_adapter[m]
//
// A negative index takes no adapter; an index past the last adapter takes none either and sets
// DEVERR_BOUNDS in the device error word.
#include <algorithm>
#include <cstring>

#include "di_common.cuh"

namespace di {

struct LoraParams {
  const void *X, *W, *A, *B, *R;
  void* Y;
  long long ldx, ldr, ldy;
  int M, N, K, r, L;
  const float *scale, *bias;
  const int* rows;
  int act;
  float* T;  // [M][r] scale[a] * X A^T
  int* err;
};

namespace {

template <typename E>
__global__ void lora_shrink_kernel(LoraParams p) {
  pdl_begin();
  const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31;
  if (i >= (long long)p.M * p.r) return;
  const int m = (int)(i / p.r), j = (int)(i % p.r);
  int a = __ldg(p.rows + m);
  if (a >= p.L) {
    if (lane == 0 && j == 0) atomicOr(p.err, DEVERR_BOUNDS);
    a = -1;
  }
  float s = 0.f;
  if (a >= 0) {
    const E* x = static_cast<const E*>(p.X) + m * p.ldx;
    const E* w = static_cast<const E*>(p.A) + ((long long)a * p.r + j) * p.K;
    for (int k = lane; k < p.K; k += 32) s = fmaf(to_f(x[k]), to_f(w[k]), s);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= __ldg(p.scale + a);
  }
  if (lane == 0) p.T[i] = s;
}

template <typename E>
__global__ void lora_expand_kernel(LoraParams p) {
  pdl_begin();
  __shared__ float xs[16][33], ws[16][33];
  const int n = blockIdx.x * 16 + threadIdx.x, m = blockIdx.y * 16 + threadIdx.y;
  const int tid = threadIdx.y * 16 + threadIdx.x;
  float s = 0.f;
  for (int k0 = 0; k0 < p.K; k0 += 32) {
    for (int q = tid; q < 512; q += 256) {
      const int rr = q / 32, kk = q % 32;
      const int mm = blockIdx.y * 16 + rr, nn = blockIdx.x * 16 + rr;
      xs[rr][kk] = mm < p.M ? to_f(static_cast<const E*>(p.X)[mm * p.ldx + k0 + kk]) : 0.f;
      ws[rr][kk] = nn < p.N ? to_f(static_cast<const E*>(p.W)[(long long)nn * p.K + k0 + kk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 32; ++kk) s = fmaf(xs[threadIdx.y][kk], ws[threadIdx.x][kk], s);
    __syncthreads();
  }
  if (m >= p.M || n >= p.N) return;
  if (p.bias) s += p.bias[n];
  const int a = p.rows[m];
  if (a >= 0 && a < p.L)
    for (int j = 0; j < p.r; ++j)
      s = fmaf(p.T[(long long)m * p.r + j], to_f(static_cast<const E*>(p.B)[((long long)a * p.N + n) * p.r + j]), s);
  if (p.act == 1) s = silu_f(s);
  else if (p.act == 2) s = gelu_erf(s);
  if (p.R) s += to_f(static_cast<const E*>(p.R)[m * p.ldr + n]);
  static_cast<E*>(p.Y)[m * p.ldy + n] = from_f<E>(s);
}

}  // namespace
}  // namespace di

using namespace di;

extern "C" size_t di_linear_lora_workspace(di_ctx_t h, int M, int N, int K, int rank, int n_adapters) {
  if (!h || M <= 0 || rank <= 0) return 0;
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
  const size_t need = di_linear_lora_workspace(h, M, N, K, rank, n_adapters);
  if (need && (!ws || ws_bytes < need || !aligned16(ws)))
    return set_error(c, DI_EINVAL, "linear_lora: workspace missing, too small or not 16-byte aligned");
  LoraParams p = {X, W, A, B, R, Y, ldx, ldr, ldy, M, N, K, rank, n_adapters, scale, bias, row_adapter, act,
                  static_cast<float*>(ws), c->d_err};
  const dim3 g1((unsigned)(((long long)M * rank * 32 + 255) / 256)), g2((N + 15) / 16, (M + 15) / 16);
  if (dtype == DI_F16) {
    launch_k(lora_shrink_kernel<__half>, g1, 256, 0, c->stream, p);
    launch_k(lora_expand_kernel<__half>, g2, dim3(16, 16), 0, c->stream, p);
  } else {
    launch_k(lora_shrink_kernel<__nv_bfloat16>, g1, 256, 0, c->stream, p);
    launch_k(lora_expand_kernel<__nv_bfloat16>, g2, dim3(16, 16), 0, c->stream, p);
  }
  return check_launch(c, "linear_lora");
}
