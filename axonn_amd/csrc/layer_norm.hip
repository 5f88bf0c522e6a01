// Layer norm over the rows of a matrix (gfx950), with the residual add in front of it:
//   h = round(x + r)   (x itself without r)
//   mean = sum(h) / N,  rstd = 1 / sqrt(sum((h - mean)^2) / N + eps),  y = (h - mean) rstd w + b
// and its backward pass, xhat = (h - mean) rstd, a = dy w:
//   dx = rstd (a - sum(a) / N - xhat sum(a xhat) / N) + dsum
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
// Sums are held in fp32; the variance is that of the deviations from the mean, not a difference
// of two sums, so that rows far from zero keep theirs.  dw and db are added up in fp32 in a
// fixed order: per workgroup, then over the workgroups' partial sums in a second launch.
#include "axn_internal.h"

namespace axn {
namespace {

template <int DT> struct Elem;
template <> struct Elem<AXN_BF16> {
  typedef __bf16 type;
};
template <> struct Elem<AXN_F16> {
  typedef _Float16 type;
};
template <> struct Elem<AXN_F32> {
  typedef float type;
};

// Parameters come in the activations' type or in fp32.
template <typename T>
__device__ __forceinline__ float param_at(const void* p, int wide, int64_t i) {
  return wide ? ((const float*)p)[i] : (float)((const T*)p)[i];
}

constexpr int ROW_THREADS = 256;

template <int THREADS>
__device__ __forceinline__ float block_sum(float x, float* shared) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  if (THREADS == 64) return x;
  __syncthreads();   // (the sums of an earlier call have been read)
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) x += shared[w];
  return x;
}

struct NormArgs {
  const void *x, *r, *w, *b;
  void *y, *h;
  float *mean, *rstd;
  int64_t M, N, ldx, ldr;
  float eps;
  int wide;
};

// Rows of any length, element by element, one workgroup to a row.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) norm_any_kernel(const NormArgs a) {
  __shared__ float shared[ROW_THREADS / 64];
  const int64_t row = block_number();
  if (row >= a.M) return;
  const T* x = (const T*)a.x + row * a.ldx;
  const T* r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  auto at = [&](int64_t i) -> float { return r ? (float)(T)((float)x[i] + (float)r[i]) : (float)x[i]; };
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < a.N; i += ROW_THREADS) s += at(i);
  const float mean = block_sum<ROW_THREADS>(s, shared) / (float)a.N;
  s = 0.0f;
  for (int64_t i = threadIdx.x; i < a.N; i += ROW_THREADS) {
    const float d = at(i) - mean;
    s += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum<ROW_THREADS>(s, shared) / (float)a.N + a.eps);
  for (int64_t i = threadIdx.x; i < a.N; i += ROW_THREADS) {
    const float h = at(i);
    float y = (h - mean) * rstd;
    if (a.w) y *= param_at<T>(a.w, a.wide, i);
    if (a.b) y += param_at<T>(a.b, a.wide, i);
    ((T*)a.y)[row * a.N + i] = (T)y;
    if (a.h) ((T*)a.h)[row * a.N + i] = (T)h;
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

struct NormGradArgs {
  const void *dy, *h, *w, *dsum;
  const float *mean, *rstd;
  void *dx, *dw, *db;
  float* partial;        // [parts][2][N]: sums of dy xhat, sums of dy
  int64_t M, N, lddy, ldh, ldsum;
  int parts, wide;
};

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) norm_dx_any_kernel(const NormGradArgs a) {
  __shared__ float shared[ROW_THREADS / 64];
  const int64_t row = block_number();
  if (row >= a.M) return;
  const T* dy = (const T*)a.dy + row * a.lddy;
  const T* h = (const T*)a.h + row * a.ldh;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t i = threadIdx.x; i < a.N; i += ROW_THREADS) {
    const float g = (float)dy[i] * (a.w ? param_at<T>(a.w, a.wide, i) : 1.0f);
    s1 += g;
    s2 += g * (((float)h[i] - mean) * rstd);
  }
  s1 = block_sum<ROW_THREADS>(s1, shared) / (float)a.N;
  s2 = block_sum<ROW_THREADS>(s2, shared) / (float)a.N;
  for (int64_t i = threadIdx.x; i < a.N; i += ROW_THREADS) {
    const float g = (float)dy[i] * (a.w ? param_at<T>(a.w, a.wide, i) : 1.0f);
    float d = (g - s1 - ((float)h[i] - mean) * rstd * s2) * rstd;
    if (a.dsum) d += (float)((const T*)a.dsum)[row * a.ldsum + i];
    ((T*)a.dx)[row * a.N + i] = (T)d;
  }
}

// Column sums of dy xhat and dy over the rows of one part: a thread to a column.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) norm_dparam_any_kernel(const NormGradArgs a) {
  const int64_t col = block_number() * ROW_THREADS + threadIdx.x;
  if (col >= a.N) return;
  const int part = blockIdx.z;
  const int64_t first = a.M * part / a.parts, last = a.M * (part + 1) / a.parts;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = first; row < last; ++row) {
    const float g = (float)((const T*)a.dy)[row * a.lddy + col];
    dw += g * (((float)((const T*)a.h)[row * a.ldh + col] - a.mean[row]) * a.rstd[row]);
    db += g;
  }
  a.partial[(int64_t)part * 2 * a.N + col] = dw;
  a.partial[((int64_t)part * 2 + 1) * a.N + col] = db;
}

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) norm_dparam_sum_kernel(const NormGradArgs a) {
  const int64_t col = block_number() * ROW_THREADS + threadIdx.x;
  if (col >= a.N) return;
  float dw = 0.0f, db = 0.0f;
  for (int part = 0; part < a.parts; ++part) {
    dw += a.partial[(int64_t)part * 2 * a.N + col];
    db += a.partial[((int64_t)part * 2 + 1) * a.N + col];
  }
  if (a.dw) {
    if (a.wide) ((float*)a.dw)[col] = dw; else ((T*)a.dw)[col] = (T)dw;
  }
  if (a.db) {
    if (a.wide) ((float*)a.db)[col] = db; else ((T*)a.db)[col] = (T)db;
  }
}

template <int DT>
int norm_launch(const NormArgs& a, hipStream_t stream) {
  typedef typename Elem<DT>::type T;
  hipLaunchKernelGGL(norm_any_kernel<T>, grid_of(a.M), dim3(ROW_THREADS), 0, stream, a);
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

template <int DT>
int norm_grad_launch(const NormGradArgs& a, hipStream_t stream) {
  typedef typename Elem<DT>::type T;
  if (a.dx) {
    hipLaunchKernelGGL(norm_dx_any_kernel<T>, grid_of(a.M), dim3(ROW_THREADS), 0, stream, a);
    AXN_HIP_TRY(hipGetLastError());
  }
  if (a.dw || a.db) {
    dim3 grid = grid_of(ceil_div(a.N, ROW_THREADS));
    if (a.parts > 0) {   // (no rows: sums of nothing)
      dim3 all = grid;
      all.z = a.parts;
      hipLaunchKernelGGL(norm_dparam_any_kernel<T>, all, dim3(ROW_THREADS), 0, stream, a);
      AXN_HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(norm_dparam_sum_kernel<T>, grid, dim3(ROW_THREADS), 0, stream, a);
    AXN_HIP_TRY(hipGetLastError());
  }
  return AXN_OK;
}

// Into how many parts the rows are cut for the sums over them.
int norm_grad_parts(int64_t M) {
  const int64_t parts = ceil_div(M, 16);
  return parts > 256 ? 256 : (int)parts;
}

}  // namespace

size_t layer_norm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M < 1 || N < 1) return 0;
  return (size_t)norm_grad_parts(M) * 2 * (size_t)N * sizeof(float);
}

int launch_layer_norm_fwd(const void* x, const void* r, const void* w, const void* b, void* y, void* h, float* mean,
                          float* rstd, int dtype, bool wide, int64_t M, int64_t N, int64_t ldx, int64_t ldr, float eps,
                          hipStream_t stream) {
  const NormArgs a = {x, r, w, b, y, h, mean, rstd, M, N, ldx, ldr, eps, wide};
  switch (dtype) {
    case AXN_BF16: return norm_launch<AXN_BF16>(a, stream);
    case AXN_F16: return norm_launch<AXN_F16>(a, stream);
    default: return norm_launch<AXN_F32>(a, stream);
  }
}

int launch_layer_norm_bwd(const void* dy, const void* h, const void* w, const float* mean, const float* rstd,
                          const void* dsum, void* dx, void* dw, void* db, int dtype, bool wide, int64_t M, int64_t N,
                          int64_t lddy, int64_t ldh, int64_t ldsum, void* ws, hipStream_t stream) {
  const NormGradArgs a = {dy, h, w, dsum, mean, rstd, dx, dw, db, (float*)ws, M, N, lddy, ldh, ldsum,
                          norm_grad_parts(M), wide};
  switch (dtype) {
    case AXN_BF16: return norm_grad_launch<AXN_BF16>(a, stream);
    case AXN_F16: return norm_grad_launch<AXN_F16>(a, stream);
    default: return norm_grad_launch<AXN_F32>(a, stream);
  }
}

}  // namespace axn
