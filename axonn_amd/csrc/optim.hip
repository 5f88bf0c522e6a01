// Mixed-precision optimizer step for gfx950 (MI355X): multi-tensor, HBM
// streaming.  Three kernels share one addressing scheme:
//   mt_scan   one read pass over the low-precision gradients: overflow check
//             (axonn/inter_layer.py:435-445) + sum of squares of the unscaled
//             gradients (axonn/intra_layer/gradient_normalization.py:18-34)
//   mt_adam   one read-modify-write pass: unscale, clip, Adam on the fp32
//             master weights and moments, low-precision copy of the weights
//             (axonn/optim.py:157-190)
//   mt_scale  in-place scaling of the gradients
//             (axonn/inter_layer.py:458, gradient_normalization.py:88-93)
// The addressing of their tensors and the update's way through memory: multi_tensor.h.
#include "axn_internal.h"
#include "multi_tensor.h"

#include <cmath>
#include <mutex>

namespace axn {
namespace {

constexpr int MT_THREADS = 256;    // threads per workgroup
constexpr int MT_VEC = 8;          // elements per lane per step
// Elements per workgroup.  The read-only scan streams best in long runs with
// non-temporal loads, measured on MI355X.
constexpr int SCAN_CHUNK = 65536;
constexpr int SCALE_CHUNK = 16384;
// Memory access policies, compile-time per call site.
template <bool NT, typename T>
__device__ __forceinline__ T ld(const T* p) {
  if (NT) return __builtin_nontemporal_load(p);
  return *p;
}
template <bool NT, typename T>
__device__ __forceinline__ void st(T v, T* p) {
  if (NT) __builtin_nontemporal_store(v, p); else *p = v;
}

struct ScanPartial {
  float sumsq;
  float sum;
  int32_t nonfinite;
  int32_t pad;
};

// 8 consecutive low-precision elements from a 16-byte aligned address.
template <int DT, bool NT>
__device__ __forceinline__ void load8(const void* base, int64_t i,
                                      typename Lowp<DT>::raw (&r)[8]) {
  typedef typename Lowp<DT>::raw raw;
  const raw* p = (const raw*)base + i;
  if (sizeof(raw) == 2) {
    const u32x4 w = ld<NT>((const u32x4*)p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[2 * e] = (raw)(w[e] & 0xFFFFu);
      r[2 * e + 1] = (raw)(w[e] >> 16);
    }
  } else {
    const u32x4 w0 = ld<NT>((const u32x4*)p);
    const u32x4 w1 = ld<NT>((const u32x4*)p + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[e] = (raw)w0[e];
      r[4 + e] = (raw)w1[e];
    }
  }
}

template <int DT, bool NT>
__device__ __forceinline__ void store8(void* base, int64_t i,
                                       const typename Lowp<DT>::raw (&r)[8]) {
  typedef typename Lowp<DT>::raw raw;
  raw* p = (raw*)base + i;
  if (sizeof(raw) == 2) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = (uint32_t)r[2 * e] | ((uint32_t)r[2 * e + 1] << 16);
    st<NT>(w, (u32x4*)p);
  } else {
    u32x4 w0, w1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w0[e] = (uint32_t)r[e];
      w1[e] = (uint32_t)r[4 + e];
    }
    st<NT>(w0, (u32x4*)p);
    st<NT>(w1, (u32x4*)p + 1);
  }
}

template <bool NT>
__device__ __forceinline__ void loadf8(const float* p, float (&x)[8]) {
  const f32x4 a = ld<NT>((const f32x4*)p);
  const f32x4 b = ld<NT>((const f32x4*)p + 1);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = a[e];
    x[4 + e] = b[e];
  }
}
template <bool NT>
__device__ __forceinline__ void storef8(float* p, const float (&x)[8]) {
  f32x4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
  st<NT>(a, (f32x4*)p);
  st<NT>(b, (f32x4*)p + 1);
}

// ---------------------------------------------------------------- scan ------
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}
__device__ __forceinline__ int wave_or(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x |= __shfl_xor(x, o, 64);
  return x;
}

// |u|^p of the norm's order p, by mode: the 2-norm and the 1-norm have their own
// instructions, order 0 counts the non-zero elements (torch.norm's meaning of p = 0),
// any other order goes through exp2(p log2 |u|) (|0|^p is 0 for p > 0 and +inf for p < 0,
// as in torch).
// Orders +inf and -inf are the largest and the smallest |u|: their terms are combined by
// max / min instead of a sum, a NaN staying a NaN as in torch.
enum NormMode { NORM_2 = 0, NORM_1 = 1, NORM_0 = 2, NORM_P = 3, NORM_MAX = 4, NORM_MIN = 5 };
template <int MODE>
__device__ __forceinline__ float norm_term(float u, float p) {
  if (MODE == NORM_2) return u * u;
  if (MODE == NORM_1 || MODE == NORM_MAX || MODE == NORM_MIN) return fabsf(u);
  if (MODE == NORM_0) return u != 0.0f ? 1.0f : 0.0f;
  return powf(fabsf(u), p);
}
// How two partial results of a mode meet, and the value that changes nothing.
template <int MODE, typename T>
__device__ __forceinline__ T norm_join(T a, T b) {
  if (MODE == NORM_MAX) return (a >= b || a != a) ? a : b;
  if (MODE == NORM_MIN) return (a <= b || a != a) ? a : b;
  return a + b;
}
template <int MODE>
__device__ __forceinline__ float norm_identity() {
  return MODE == NORM_MIN ? __builtin_inff() : 0.0f;
}

template <int DT, int MODE>
__global__ void __launch_bounds__(MT_THREADS)
    mt_scan_kernel(const MtTable tab, float inv_scale, float norm_type, ScanPartial* partial,
                   int block_base) {
  typedef typename Lowp<DT>::raw raw;
  const int t = find_tensor(tab, blockIdx.x);
  const int c = blockIdx.x - tab.chunk_start[t];
  const Range rg = chunk_range(tab, t, c);
  const void* g = tab.g[t];
  const int tid = threadIdx.x;

  float sq = norm_identity<MODE>(), sm = 0.f;
  int bad = 0;
  auto one = [&](raw x) {
    bad |= Lowp<DT>::nonfinite(x) ? 1 : 0;
    const float f = Lowp<DT>::to_float(x);
    sm += f;
    sq = norm_join<MODE>(sq, norm_term<MODE>(f * inv_scale, norm_type));
  };
  if (vec_ok_of(tab, t)) {
    if (c == 0 && tid < head_of(tab, t)) one(((const raw*)g)[tid]);
    const int64_t nvec = (rg.end - rg.begin) / MT_VEC;
    for (int64_t i = tid; i < nvec; i += MT_THREADS) {
      raw r[8];
      load8<DT, true>(g, rg.begin + i * MT_VEC, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) one(r[e]);
    }
    const int64_t tail = rg.begin + nvec * MT_VEC;
    if (tail + tid < rg.end) one(((const raw*)g)[tail + tid]);
  } else {
    const int64_t b = (c == 0) ? 0 : rg.begin;
    for (int64_t i = b + tid; i < rg.end; i += MT_THREADS) one(((const raw*)g)[i]);
  }

  __shared__ float s_sq[MT_THREADS / 64], s_sm[MT_THREADS / 64];
  __shared__ int s_bad[MT_THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sq = norm_join<MODE>(sq, __shfl_xor(sq, o, 64));
  sm = wave_sum(sm);
  bad = wave_or(bad);
  if ((tid & 63) == 0) {
    s_sq[tid >> 6] = sq;
    s_sm[tid >> 6] = sm;
    s_bad[tid >> 6] = bad;
  }
  __syncthreads();
  if (tid == 0) {
    ScanPartial p;
    p.sumsq = norm_identity<MODE>();
    p.sum = 0.f;
    p.nonfinite = 0;
#pragma unroll
    for (int w = 0; w < MT_THREADS / 64; ++w) {  // fixed order: deterministic
      p.sumsq = norm_join<MODE>(p.sumsq, s_sq[w]);
      p.sum += s_sm[w];
      p.nonfinite |= s_bad[w];
    }
    p.pad = 0;
    partial[block_base + blockIdx.x] = p;
  }
}

__device__ __forceinline__ double wave_sum_d(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// One workgroup of 1024 threads reduces the partials of one launch group in a
// fixed order: wave w takes tensors w, w + 16, ...; lanes stride over that
// tensor's chunks.  `first` initialises the result, later groups accumulate.
template <int MODE>
__global__ void __launch_bounds__(1024)
    mt_scan_finalize_kernel(const MtTable tab, const ScanPartial* partial,
                            int block_base, double sum_limit, float max_norm,
                            float norm_type, int first, axn_scan_result* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ double s_sq[16];
  __shared__ int s_bad[16];
  double sq = (double)norm_identity<MODE>();
  int bad = 0;
  for (int t = wave; t < tab.n; t += 16) {
    double tsq = (double)norm_identity<MODE>(), tsm = 0.0;
    int tbad = 0;
    for (int b = tab.chunk_start[t] + lane; b < tab.chunk_start[t + 1]; b += 64) {
      const ScanPartial p = partial[block_base + b];
      tsq = norm_join<MODE>(tsq, (double)p.sumsq);
      tsm += (double)p.sum;
      tbad |= p.nonfinite;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) tsq = norm_join<MODE>(tsq, __shfl_xor(tsq, o, 64));
    tsm = wave_sum_d(tsm);
    tbad = wave_or(tbad);
    // The tensor's sum, rounded to the gradient dtype, is non-finite.
    if (!(fabs(tsm) < sum_limit)) tbad = 1;
    // order 0: the norm over the stacked per-tensor norms counts the tensors whose own
    // count of non-zero elements is not zero
    if (MODE == NORM_0) tsq = tsq != 0.0 ? 1.0 : 0.0;
    sq = norm_join<MODE>(sq, tsq);
    bad |= tbad;
  }
  if (lane == 0) {
    s_sq[wave] = sq;
    s_bad[wave] = bad;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = first ? (double)norm_identity<MODE>() : out->sumsq;
    int flag = first ? 0 : out->found_inf;
    for (int w = 0; w < 16; ++w) {
      total = norm_join<MODE>(total, s_sq[w]);
      flag |= s_bad[w];
    }
    const float norm = MODE == NORM_2 ? (float)sqrt(total)
                       : MODE == NORM_P ? (float)pow(total, 1.0 / (double)norm_type)
                                        : (float)total;
    float coef = 1.0f;
    if (max_norm > 0.0f) {
      coef = max_norm / (norm + 1e-6f);
      if (coef > 1.0f) coef = 1.0f;  // a NaN coefficient stays NaN, as torch.clamp keeps it
    }
    out->sumsq = total;
    out->total_norm = norm;
    out->clip_coef = coef;
    out->found_inf = flag;
    out->reserved[0] = out->reserved[1] = out->reserved[2] = 0;
  }
}

// ---------------------------------------------------------------- adam ------
struct AdamScalars {
  axn_adam_hparams hp;
  float inv_scale;
};

__device__ __forceinline__ void adam_math(float g, float& p, float& m, float& v,
                                          const AdamScalars& s, float gmul) {
  g = g * s.inv_scale;
  g = g * gmul;
  if (s.hp.weight_decay != 0.0f) g = g + s.hp.weight_decay * p;
  m = m + (g - m) * s.hp.one_minus_beta1;
  v = v * s.hp.beta2 + s.hp.one_minus_beta2 * g * g;
  const float denom = sqrtf(v) * s.hp.inv_sqrt_bc2 + s.hp.eps;
  p = p - s.hp.lr_over_bc1 * (m / denom);
  // The low-precision copy must be the rounding of the fp32 value that is
  // stored, not of the unrounded expression: keep the compiler from folding
  // the conversion into the last multiply-add (a mixed-precision FMA rounds once).
  asm volatile("" : "+v"(p));
}

template <int GDT, int PDT, bool HAS_PLOW, bool HAS_SCAN>
__global__ void __launch_bounds__(ADAM_THREADS)
    mt_adam_kernel(const MtTable tab, const AdamScalars s, const axn_scan_result* scan) {
  const int b = blockIdx.x;
  const TensorRow row = row_by_scalar_search(tab, b);
  int found_inf = 0;
  float gmul = 1.0f;
  if (HAS_SCAN) {   // (beside the lookup, not in front of it)
    found_inf = scan->found_inf;
    gmul = scan->clip_coef;
  }
  update_chunk<GDT, PDT, HAS_PLOW>(row, b, found_inf, gmul, [&](float g, float& p, float& m, float& v, float mul) {
    adam_math(g, p, m, v, s, mul);
  });
}

// --------------------------------------------------------------- scale ------
template <int DT>
__global__ void __launch_bounds__(MT_THREADS)
    mt_scale_kernel(const MtTable tab, float inv_scale,
                    const axn_scan_result* scan, int use_clip) {
  typedef typename Lowp<DT>::raw raw;
  const float coef = use_clip ? scan->clip_coef : 1.0f;
  const int t = find_tensor(tab, blockIdx.x);
  const int c = blockIdx.x - tab.chunk_start[t];
  const Range rg = chunk_range(tab, t, c);
  void* g = const_cast<void*>(tab.g[t]);
  const int tid = threadIdx.x;
  // Two roundings, as the reference's separate div_ and mul_ passes make.
  auto f = [&](raw x) -> raw {
    raw y = Lowp<DT>::from_float(Lowp<DT>::to_float(x) * inv_scale);
    if (use_clip) y = Lowp<DT>::from_float(Lowp<DT>::to_float(y) * coef);
    return y;
  };
  if (vec_ok_of(tab, t)) {
    if (c == 0 && tid < head_of(tab, t)) ((raw*)g)[tid] = f(((raw*)g)[tid]);
    const int64_t nvec = (rg.end - rg.begin) / MT_VEC;
    for (int64_t i = tid; i < nvec; i += MT_THREADS) {
      raw r[8];
      load8<DT, false>(g, rg.begin + i * MT_VEC, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = f(r[e]);
      store8<DT, true>(g, rg.begin + i * MT_VEC, r);
    }
    const int64_t tail = rg.begin + nvec * MT_VEC;
    if (tail + tid < rg.end) ((raw*)g)[tail + tid] = f(((raw*)g)[tail + tid]);
  } else {
    const int64_t b = (c == 0) ? 0 : rg.begin;
    for (int64_t i = b + tid; i < rg.end; i += MT_THREADS) ((raw*)g)[i] = f(((raw*)g)[i]);
  }
}

// ------------------------------------------------------------- host side ----
double sum_limit_of(int dt) {
  // Smallest magnitude that rounds (to nearest even) to infinity in the dtype.
  switch (dt) {
    case AXN_F16: return 65520.0;
    case AXN_BF16: return 3.3961775292304601e38;   // 2^127 * (2 - 2^-8)
    default: return 3.4028235677973366e38;         // 2^127 * (2 - 2^-24)
  }
}

int norm_mode_host(float p) {
  return p == 2.0f ? NORM_2 : p == 1.0f ? NORM_1 : p == 0.0f ? NORM_0
         : p == INFINITY ? NORM_MAX : p == -INFINITY ? NORM_MIN : NORM_P;
}

template <int DT>
void scan_dispatch(const Group& gr, float inv_scale, float norm_type, ScanPartial* partial,
                   int base, hipStream_t stream) {
  const dim3 grid(gr.blocks), block(MT_THREADS);
  switch (norm_mode_host(norm_type)) {
#define AXN_SCAN_CASE(MODE)                                                                     \
  case MODE:                                                                                    \
    hipLaunchKernelGGL((mt_scan_kernel<DT, MODE>), grid, block, 0, stream, gr.tab, inv_scale,   \
                       norm_type, partial, base);                                               \
    break;
    AXN_SCAN_CASE(NORM_2)
    AXN_SCAN_CASE(NORM_1)
    AXN_SCAN_CASE(NORM_0)
    AXN_SCAN_CASE(NORM_MAX)
    AXN_SCAN_CASE(NORM_MIN)
    default:
    AXN_SCAN_CASE(NORM_P)
#undef AXN_SCAN_CASE
  }
}

void finalize_dispatch(const MtTable& tab, const ScanPartial* partial, int base, double sum_limit,
                       float max_norm, float norm_type, int first, axn_scan_result* result,
                       hipStream_t stream) {
  switch (norm_mode_host(norm_type)) {
#define AXN_FIN_CASE(MODE)                                                                       \
  case MODE:                                                                                     \
    hipLaunchKernelGGL(mt_scan_finalize_kernel<MODE>, dim3(1), dim3(1024), 0, stream, tab,       \
                       partial, base, sum_limit, max_norm, norm_type, first, result);            \
    break;
    AXN_FIN_CASE(NORM_2)
    AXN_FIN_CASE(NORM_1)
    AXN_FIN_CASE(NORM_0)
    AXN_FIN_CASE(NORM_MAX)
    AXN_FIN_CASE(NORM_MIN)
    default:
    AXN_FIN_CASE(NORM_P)
#undef AXN_FIN_CASE
  }
}

}  // namespace
}  // namespace axn

// Scratch of axn_mt_scan_noalloc: the per-chunk partial results of the scan, in device
// memory that exists for the life of the process (1 MiB per GPU the library runs on).
// This name is a host-side handle only; the device address is looked up per device.
static __device__ __align__(256) unsigned char scratch[AXN_MT_SCAN_SCRATCH_BYTES];

namespace axn {
namespace {

// Device address of `scratch` on the current device, looked up once per device.
int scan_scratch(void** out) {
  static std::mutex mu;
  static void* ptrs[64];
  int dev = 0;
  AXN_HIP_TRY(hipGetDevice(&dev));
  if (dev < 0 || dev >= 64) {
    set_error("axn_mt_scan_noalloc: device index %d out of range", dev);
    return AXN_ELIMIT;
  }
  std::lock_guard<std::mutex> lock(mu);
  if (ptrs[dev] == nullptr) {
    void* p = nullptr;
    AXN_HIP_TRY(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
    if (p == nullptr) {
      set_error("axn_mt_scan_noalloc: no device address for the scratch array");
      return AXN_EHIP;
    }
    ptrs[dev] = p;
  }
  *out = ptrs[dev];
  return AXN_OK;
}

}  // namespace

size_t mt_scan_workspace_bytes(int64_t n, int64_t total) {
  if (n < 0 || total < 0) return 0;
  // One partial per chunk; a tensor adds at most one ragged chunk.
  const int64_t blocks = total / SCAN_CHUNK + 2 * n + 1;
  return (size_t)blocks * sizeof(ScanPartial);
}

int launch_mt_scan(const void* const* h_g, const int64_t* h_sizes, int64_t n,
                   int g_dtype, float inv_scale, float max_norm, float norm_type,
                   int accumulate, axn_scan_result* result, void* ws, size_t ws_bytes,
                   hipStream_t stream) {
  const void* const* sets[1] = {h_g};
  const int es[1] = {dtype_size(g_dtype)};
  // first walk: what the partial results need
  int64_t need = 0;
  int rc = for_each_group(sets, es, 1, h_sizes, n, SCAN_CHUNK, MT_THREADS, [&](const Group& gr) {
    need += gr.blocks;
    return (int)AXN_OK;
  });
  if (rc != AXN_OK) return rc;
  if ((size_t)need * sizeof(ScanPartial) > ws_bytes) {
    set_error("mt_scan: workspace too small (%zu bytes given, %zu needed)",
              ws_bytes, (size_t)need * sizeof(ScanPartial));
    return AXN_EINVAL;
  }
  ScanPartial* partial = (ScanPartial*)ws;
  if (need == 0) {
    // Nothing to scan: norm 0, no overflow.
    MtTable empty = MtTable();
    empty.n = 0;
    empty.chunk = SCAN_CHUNK;
    // (nothing scanned and nothing to add to: every order's norm is 0)
    finalize_dispatch(empty, partial, 0, sum_limit_of(g_dtype), max_norm, accumulate ? norm_type : 2.0f,
                      accumulate ? 0 : 1, result, stream);
    AXN_HIP_TRY(hipGetLastError());
    return AXN_OK;
  }
  int base = 0;
  bool first = !accumulate;
  return for_each_group(sets, es, 1, h_sizes, n, SCAN_CHUNK, MT_THREADS, [&](const Group& gr) {
    switch (g_dtype) {
      case AXN_BF16: scan_dispatch<AXN_BF16>(gr, inv_scale, norm_type, partial, base, stream); break;
      case AXN_F16: scan_dispatch<AXN_F16>(gr, inv_scale, norm_type, partial, base, stream); break;
      default: scan_dispatch<AXN_F32>(gr, inv_scale, norm_type, partial, base, stream); break;
    }
    AXN_HIP_TRY(hipGetLastError());
    finalize_dispatch(gr.tab, partial, base, sum_limit_of(g_dtype), max_norm, norm_type, first ? 1 : 0,
                      result, stream);
    AXN_HIP_TRY(hipGetLastError());
    base += gr.blocks;
    first = false;
    return (int)AXN_OK;
  });
}

int launch_mt_scan_noalloc(const void* const* h_g, const int64_t* h_sizes, int64_t n,
                           int g_dtype, float inv_scale, float max_norm, float norm_type,
                           int accumulate, axn_scan_result* result, hipStream_t stream) {
  // the size limit is checked before anything touches the device
  const void* const* sets[1] = {h_g};
  const int es[1] = {dtype_size(g_dtype)};
  int64_t need = 0;
  int rc = for_each_group(sets, es, 1, h_sizes, n, SCAN_CHUNK, MT_THREADS, [&](const Group& gr) {
    need += gr.blocks;
    return (int)AXN_OK;
  });
  if (rc != AXN_OK) return rc;
  if ((size_t)need * sizeof(ScanPartial) > (size_t)AXN_MT_SCAN_SCRATCH_BYTES) {
    set_error("axn_mt_scan_noalloc: the gradients make %lld chunks of %d elements, the built-in "
              "scratch holds %lld; use axn_mt_scan with a workspace",
              (long long)need, SCAN_CHUNK,
              (long long)(AXN_MT_SCAN_SCRATCH_BYTES / sizeof(ScanPartial)));
    return AXN_ELIMIT;
  }
  void* ws = nullptr;
  rc = scan_scratch(&ws);
  if (rc != AXN_OK) return rc;
  return launch_mt_scan(h_g, h_sizes, n, g_dtype, inv_scale, max_norm, norm_type, accumulate,
                        result, ws, (size_t)AXN_MT_SCAN_SCRATCH_BYTES, stream);
}

namespace {
template <int GDT, bool HAS_SCAN>
int adam_launch(const Group& gr, const AdamScalars& s, int plow_dtype, bool has_plow,
                const axn_scan_result* scan, hipStream_t stream) {
  const dim3 grid((unsigned)gr.blocks), block(ADAM_THREADS);
  if (!has_plow) {
    hipLaunchKernelGGL((mt_adam_kernel<GDT, AXN_BF16, false, HAS_SCAN>), grid, block, ADAM_LDS,
                       stream, gr.tab, s, scan);
  } else if (plow_dtype == AXN_BF16) {
    hipLaunchKernelGGL((mt_adam_kernel<GDT, AXN_BF16, true, HAS_SCAN>), grid, block, ADAM_LDS,
                       stream, gr.tab, s, scan);
  } else {
    hipLaunchKernelGGL((mt_adam_kernel<GDT, AXN_F16, true, HAS_SCAN>), grid, block, ADAM_LDS,
                       stream, gr.tab, s, scan);
  }
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}
template <int GDT>
int adam_dispatch(const Group& gr, const AdamScalars& s, int plow_dtype,
                  bool has_plow, const axn_scan_result* scan, hipStream_t stream) {
  return scan != nullptr ? adam_launch<GDT, true>(gr, s, plow_dtype, has_plow, scan, stream)
                         : adam_launch<GDT, false>(gr, s, plow_dtype, has_plow, scan, stream);
}
}  // namespace

int launch_mt_adam(const void* const* h_g, void* const* h_p, void* const* h_m,
                   void* const* h_v, void* const* h_plow, const int64_t* h_sizes,
                   int64_t n, int g_dtype, int plow_dtype, float inv_scale,
                   const axn_scan_result* scan, const axn_adam_hparams& hp,
                   hipStream_t stream) {
  const void* const* sets[5] = {h_g, (const void* const*)h_p, (const void* const*)h_m,
                                (const void* const*)h_v, (const void* const*)h_plow};
  const int es[5] = {dtype_size(g_dtype), 4, 4, 4, dtype_size(plow_dtype)};
  AdamScalars s;
  s.hp = hp;
  s.inv_scale = inv_scale;
  const bool has_plow = h_plow != nullptr;
  return for_each_group(sets, es, 5, h_sizes, n, ADAM_CHUNK, ADAM_THREADS, [&](const Group& gr) {
    switch (g_dtype) {
      case AXN_BF16: return adam_dispatch<AXN_BF16>(gr, s, plow_dtype, has_plow, scan, stream);
      case AXN_F16: return adam_dispatch<AXN_F16>(gr, s, plow_dtype, has_plow, scan, stream);
      default: return adam_dispatch<AXN_F32>(gr, s, plow_dtype, has_plow, scan, stream);
    }
  });
}

int launch_mt_scale(void* const* h_g, const int64_t* h_sizes, int64_t n,
                    int g_dtype, float inv_scale, const axn_scan_result* scan,
                    int use_clip, hipStream_t stream) {
  const void* const* sets[1] = {(const void* const*)h_g};
  const int es[1] = {dtype_size(g_dtype)};
  return for_each_group(sets, es, 1, h_sizes, n, SCALE_CHUNK, MT_THREADS, [&](const Group& gr) {
    const dim3 grid(gr.blocks), block(MT_THREADS);
    switch (g_dtype) {
      case AXN_BF16:
        hipLaunchKernelGGL(mt_scale_kernel<AXN_BF16>, grid, block, 0, stream,
                           gr.tab, inv_scale, scan, use_clip);
        break;
      case AXN_F16:
        hipLaunchKernelGGL(mt_scale_kernel<AXN_F16>, grid, block, 0, stream,
                           gr.tab, inv_scale, scan, use_clip);
        break;
      default:
        hipLaunchKernelGGL(mt_scale_kernel<AXN_F32>, grid, block, 0, stream,
                           gr.tab, inv_scale, scan, use_clip);
        break;
    }
    AXN_HIP_TRY(hipGetLastError());
    return (int)AXN_OK;
  });
}

}  // namespace axn
