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

constexpr int64_t kL2 = 32 << 20;        // bytes that the eight L2s hold
// Bytes that the memory-side cache holds.  A forward with a residual that moves more keeps nothing in the
// caches, in two turns a workgroup: 16384 x 8192 bf16 203 -> 181 us on the same rows again and again (187 on
// others every time), with the product that reads it 368 -> 374 (8192 x 8192 215 -> 206, 32768 x 8192 753 -> 739).  Without a residual there is nothing in it (98 us
// -> 105, 279 -> 299).
constexpr int64_t kCached = 256 << 20;
constexpr int MOST_PARTS = 256;   // parts of the rows whose column sums meet in a second launch

struct NormArgs {
  const void *x, *r, *w, *b;
  void *y, *h;
  float *mean, *rstd;
  int64_t M, N, ldx, ldr;
  float eps;
  int wide, through;
};

struct NormGradArgs {
  const void *dy, *h, *w, *dsum;
  const float *mean, *rstd;
  void *dx, *dw, *db;
  float* partial;        // [parts][2][N]: sums of dy xhat, sums of dy
  int64_t M, N, lddy, ldh, ldsum;
  int parts, wide;
};

// ---------------------------------------------------------- vector kernels --
// Both passes are bound by memory: a row's elements are read once and written once.  A copy on the
// same GPU moves 6.8 TB/s; the forward moves 5.1 to 5.9 TB/s of bf16 from 20 MB on, the backward 4 to
// 5.5 (see there).
// A row lies in the registers of 16 lanes or of several whole waves, K vectors of 16 bytes in a
// lane, and is read once.  With four of them, rows of 16385 to 32768 16-bit elements, 128 registers do not
// hold it all: the forward with a residual spills 36 to 84 bytes a lane, the backward 148 to 224 (fp32,
// 8193 to 16384 elements: 16 to 24 with dsum; two vectors of 16 lanes with dsum: 12 to 20).
// Vector v of a row holds its elements from v VEC on, but the last one ends with the row and
// overlaps the one before: `twice` of its elements are in both, count once in sums and are
// stored by both with one value.  Rows may start anywhere: the accesses are declared to be
// aligned to an element only, which gfx950 reads in one instruction all the same.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef T Type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
// NT: not to be kept in the caches.
template <bool NT = false, typename T>
__device__ __forceinline__ typename Vec<T>::Type load_vec(const T* p) {
  if (NT) return __builtin_nontemporal_load((const typename Vec<T>::Type*)p);
  return *(const typename Vec<T>::Type*)p;
}
template <bool NT = false, typename T>
__device__ __forceinline__ void store_vec(T* p, typename Vec<T>::Type v) {
  if (NT)
    __builtin_nontemporal_store(v, (typename Vec<T>::Type*)p);
  else
    *(typename Vec<T>::Type*)p = v;
}
// A vector of the forward's results.  Those of a call that the L2s can hold (`through`) are written
// through them, or they are all written back when the kernel ends: 1024 x 4096 bf16 5.6 -> 4.8 us, with
// the product that reads it 20.7 -> 19.8; 3001 x 1025 fp32 7.1 -> 5.8.  From 64 MB on there is nothing in
// it (8192 x 8192 and its product 153 -> 164), and in the backward, with its second launch, little
// (1000 x 4096 15.3 -> 14.9, 16384 x 5120 99 -> 100).
// Results that bypass the caches take another 2 to 20 % less here and cost their reader more than that
// (4096 x 4096 and its product 46 -> 54 us, 8192 x 8192 154 -> 169): not done (see kCached for the exception).
template <bool NT, typename T>
__device__ __forceinline__ void store_result(T* p, typename Vec<T>::Type v, int through) {
  if (NT || !through) {
    store_vec<NT>(p, v);
  } else {
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(v) : "memory");
  }
}
// VEC parameters from element i on, as floats.
template <typename T>
__device__ __forceinline__ void load_params(const void* p, int wide, int64_t i, float (&out)[Vec<T>::N]) {
  constexpr int N = Vec<T>::N;
  if (sizeof(T) == 4 || wide) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const auto v = load_vec((const float*)p + i + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * j + e] = v[e];
    }
  } else {
    const auto v = load_vec((const T*)p + i);
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = (float)v[e];
  }
}

// Where vector v of rows of n elements starts, and how many of its elements others have.  A
// vector behind the row is its last one again, none of its elements its own, so that loads need
// no branch around them, which would have each wait for the one before.
struct Span {
  int first, twice;
};
template <int VEC>
__device__ __forceinline__ Span span_of(int v, int n) {
  const int first = min(v * VEC, n - VEC);
  return {first, min(v * VEC - first, VEC)};
}

// The same for rows of up to 2^31 - 1 elements, a vector of the row itself.
template <int VEC>
__device__ __forceinline__ Span long_span(int v, int n) {
  const int64_t end = ((int64_t)v + 1) * VEC;
  return end <= n ? Span{v * VEC, 0} : Span{n - VEC, (int)(end - n)};
}

// The threads of a row: SUB: 16 lanes, else `waves` whole waves (16 at most).
template <bool SUB>
struct RowOf {
  int waves, lane, threads, group;   // waves of a row, this thread's place among its row's, their number, the row in the workgroup
  __device__ __forceinline__ RowOf(int w) : waves(w) {
    threads = SUB ? 16 : waves * 64;
    // (the row of a whole wave is a scalar: addresses are a scalar base and a lane's offset)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    group = SUB ? (int)threadIdx.x >> 4 : wave / waves;
    lane = SUB ? (int)threadIdx.x & 15 : (wave - group * waves) * 64 + ((int)threadIdx.x & 63);
  }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// The sum over 16 neighbouring lanes, or over the wave, in all of them: rotations by 8, 4, 2
// and 1 within the rows of 16 lanes, which no LDS access or wait is behind.
__device__ __forceinline__ float row16_sum(float x) {
  x = dpp_add<0x128>(x);
  x = dpp_add<0x124>(x);
  x = dpp_add<0x122>(x);
  return dpp_add<0x121>(x);
}
__device__ __forceinline__ float lane_of(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}
__device__ __forceinline__ float wave64_sum(float x) {
  x = row16_sum(x);
  return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}
// COUNT sums over the threads of a row; the waves of one meet in `shared`, COUNT places for every
// wave, which is not written again before the next barrier but one.
template <bool SUB, int COUNT>
__device__ __forceinline__ void row_sums(float (&x)[COUNT], const RowOf<SUB>& at, float (*shared)[16]) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) x[i] = SUB ? row16_sum(x[i]) : wave64_sum(x[i]);
  if (SUB || at.waves == 1) return;
  const int lane = threadIdx.x & 63;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) shared[i][threadIdx.x >> 6] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const float mine = shared[i][at.group * at.waves + min(lane & 15, at.waves - 1)];
    x[i] = row16_sum((lane & 15) < at.waves ? mine : 0.0f);
  }
}

// The next row is on its way while one is summed.  Twice as many workgroups as are resident half full
// measured 5 to 8 % slower, half as many up to 13 % (most in norm_rows_launch).
// RES: a residual is added.  RAGGED: N is no multiple of a vector.  A workgroup takes `rows` rows at
// a time and goes on to those gridDim.x workgroups further, the parameters of its columns in
// registers; STREAM: nothing is kept in the caches.
template <typename T, int K, bool SUB, bool RES, bool RAGGED, bool STREAM>
__global__ void __launch_bounds__(1024) norm_rows_kernel(const NormArgs a, int waves, int rows) {
  constexpr int VEC = Vec<T>::N;
  typedef typename Vec<T>::Type V;
  __shared__ float shared[2][2][16];
  const RowOf<SUB> at(waves);
  const int n = (int)a.N;
  struct Row {
    V x[K], r[RES ? K : 1];
  };
  auto fetch = [&](Row& f, int64_t row) {   // (behind the last row: that row again)
    row = row < a.M ? row : a.M - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = span_of<VEC>(k * at.threads + at.lane, n).first;
      f.x[k] = load_vec<STREAM>((const T*)a.x + row * a.ldx + first);
      if (RES) f.r[k] = load_vec<STREAM>((const T*)a.r + row * a.ldr + first);
    }
  };
  const int64_t stride = (int64_t)gridDim.x * rows;
  int64_t begin = (int64_t)blockIdx.x * rows;   // the workgroup's first row of this turn
  constexpr bool AHEAD = K <= 2;
  Row one, other;
  if (AHEAD) fetch(one, begin + at.group);
  float w[K][VEC], b[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int first = span_of<VEC>(k * at.threads + at.lane, n).first;
    if (a.w) load_params<T>(a.w, a.wide, first, w[k]);
    if (a.b) load_params<T>(a.b, a.wide, first, b[k]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (!a.w) w[k][e] = 1.0f;
      if (!a.b) b[k][e] = 0.0f;
    }
  }
  int turn = 0;
  // One turn: the next one's rows are on their way while this one's are summed, if registers
  // hold both.
  auto step = [&](Row& f, Row& next) -> bool {
    const int64_t row = begin + at.group;
    const bool live = row < a.M, more = begin + stride < a.M;
    if (!AHEAD) fetch(f, row);
    if (AHEAD && more) fetch(next, row + stride);
    float h[K][VEC], s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Span span = span_of<VEC>(k * at.threads + at.lane, n);
      if (RES) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f.x[k][e] = (T)((float)f.x[k][e] + (float)f.r[k][e]);
        if (live && span.twice < VEC) store_result<STREAM>((T*)a.h + row * a.N + span.first, f.x[k], a.through);
      }
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        h[k][e] = (float)f.x[k][e];
        t += RAGGED && e < span.twice ? 0.0f : h[k][e];
      }
      s[0] += !RAGGED && span.twice ? 0.0f : t;
    }
    row_sums<SUB>(s, at, &shared[turn][0]);
    const float mean = s[0] / (float)n;   // (of equal elements, that element)
    s[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Span span = span_of<VEC>(k * at.threads + at.lane, n);
      float t = 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        h[k][e] -= mean;
        t += RAGGED && e < span.twice ? 0.0f : h[k][e] * h[k][e];
      }
      s[0] += !RAGGED && span.twice ? 0.0f : t;
    }
    row_sums<SUB>(s, at, &shared[turn][1]);
    const float rstd = 1.0f / sqrtf(s[0] / (float)n + a.eps);
    if (live) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const Span span = span_of<VEC>(k * at.threads + at.lane, n);
        if (span.twice == VEC) continue;
        V y;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float f = h[k][e] * rstd * w[k][e] + b[k][e];
          // (rounded to fp32 first with and without a residual: a mixed-precision multiply-add,
          // which the compiler takes where it likes, would round once and give other bits)
          asm volatile("" : "+v"(f));
          y[e] = (T)f;
        }
        store_result<STREAM>((T*)a.y + row * a.N + span.first, y, a.through);
      }
      if (at.lane == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
    begin += stride;
    turn ^= 1;
    return more;
  };
  if (AHEAD) {
    while (step(one, other) && step(other, one)) {
    }
  } else {
    while (step(one, one)) {
    }
  }
}

// Waves and vectors of a lane for rows of N elements, and whether 16 lanes do.  `single`: one vector
// to a lane as long as 16 waves hold the row, which the backward takes: its sums of columns then take
// half the registers (bf16 4096 x 4096 28.9 -> 27.0 us, 16384 x 5120 104 -> 99.5).  The forward, which
// has none, is faster with two (4096 x 4096 13.1 us, 15.7 with one; 8192 x 5120 33, 45).
struct RowPlan {
  int k, waves;
  bool sub;
};
inline RowPlan plan_row(int64_t N, int vec, bool single) {
  const int64_t v = ceil_div(N, vec);
  if (v <= 32) return {v <= 16 ? 1 : 2, 1, true};
  if (single && v <= 1024) return {1, (int)ceil_div(v, 64), false};
  if (v <= 2048) return {2, (int)ceil_div(v, 128), false};
  return {4, (int)ceil_div(v, 256), false};
}

template <typename T, int K, bool SUB>
int norm_rows_launch(const NormArgs& a, const RowPlan& plan, hipStream_t queue) {
  const int rows = SUB ? 16 : plan.waves >= 4 ? 1 : 4 / plan.waves;
  const int threads = SUB ? 256 : plan.waves * rows * 64;
  const bool stream = a.r && 4 * a.M * a.N * (int64_t)sizeof(T) > kCached;
  int64_t groups = ceil_div(a.M, rows);
  const int64_t most = stream ? (groups + 1) / 2 : 256 * (2048 / threads) / 2;
  if (groups > most) groups = most;
  if (groups > kMostBlocks) groups = kMostBlocks;
  const bool ragged = a.N % Vec<T>::N != 0;
#define AXN_NORM(RES, RAGGED, STREAM)                                                                              \
  if ((a.r != nullptr) == RES && ragged == RAGGED && stream == STREAM)                                             \
  hipLaunchKernelGGL((norm_rows_kernel<T, K, SUB, RES, RAGGED, STREAM>), dim3((unsigned)groups), dim3(threads), 0, \
                     queue, a, plan.waves, rows)
  AXN_NORM(false, false, false);
  AXN_NORM(false, true, false);
  AXN_NORM(true, false, false);
  AXN_NORM(true, false, true);
  AXN_NORM(true, true, false);
  AXN_NORM(true, true, true);
#undef AXN_NORM
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

template <typename T>
int norm_rows(const NormArgs& a, hipStream_t stream) {
  const RowPlan plan = plan_row(a.N, Vec<T>::N, false);
  if (plan.sub) return plan.k == 1 ? norm_rows_launch<T, 1, true>(a, plan, stream) : norm_rows_launch<T, 2, true>(a, plan, stream);
  if (plan.k == 2) return norm_rows_launch<T, 2, false>(a, plan, stream);
  return norm_rows_launch<T, 4, false>(a, plan, stream);
}

// Backward.  Its time is 11 us and the bytes at 5.7 TB/s: 3 us to launch and to the first rows, 3 for
// the workgroups' sums (8 MB of them for 4096 columns, written at the end), 4 to 5 for the second launch
// that adds them up.  256 workgroups of up to 16 waves, one to a CU, are a compromise: 512 of half the
// size, two to a CU, are 5 % faster up to their sums and 5 to 15 % slower with twice as many of those.
// 4096 x 4096 bf16 with dsum 32.7 us (4.1 TB/s), 16384 x 5120 98 us (5.1), 32768 x 4096 147 us (5.5).
// Wider rows fill a CU with one workgroup and its partial sums grow: 16384 x 8192 bf16 149 us (5.4), 8192 x
// 16384 160 us (5.0), 16384 x 8192 fp32 295 us (5.5).  Four vectors to a lane, which spill, fall off:
// 4096 x 24576 bf16 222 us (2.7), 4096 x 32768 286 us (2.8), 600 x 32768 86 us, where the kernels of long
// rows take 335 and 54 us for eight elements more; 4096 x 16384 fp32 162 us (5.0), and 313 for four more.
// Rows as above, several at a time in a workgroup, which goes on to the rows `parts`
// workgroups further until there are none.  Its threads keep the sums of dy xhat and dy of their
// columns in registers; at the end the workgroup's rows are joined in LDS and its sums go to
// `partial`.  RAGGED: N is no multiple of a vector.  SUM: dsum is given.
template <typename T, int K, bool SUB, bool RAGGED, bool SUM>
__global__ void __launch_bounds__(1024) norm_grad_rows_kernel(const NormGradArgs a, int waves, int rows) {
  constexpr int VEC = Vec<T>::N;
  typedef typename Vec<T>::Type V;
  __shared__ float meet[2][2][16];
  extern __shared__ __align__(16) float joined[];   // [rows][dw, db][vectors of a row][VEC]
  const RowOf<SUB> at(waves);
  const int n = (int)a.N;
  const float inv_n = 1.0f / (float)n;
  struct Row {
    V dy[K], h[K];
    float mean, rstd;
  };
  auto fetch = [&](Row& r, int64_t row) {   // (behind the last row: that row again, counted as nothing)
    row = row < a.M ? row : a.M - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = span_of<VEC>(k * at.threads + at.lane, n).first;
      r.dy[k] = load_vec((const T*)a.dy + row * a.lddy + first);
      r.h[k] = load_vec((const T*)a.h + row * a.ldh + first);
    }
    r.mean = a.mean[row];
    r.rstd = a.rstd[row];
  };
  const int64_t stride = (int64_t)a.parts * rows;
  int64_t begin = (int64_t)blockIdx.x * rows;   // the workgroup's first row of this turn
  constexpr bool AHEAD = K <= 2;
  Row one, other;
  if (AHEAD) fetch(one, begin + at.group);
  float w[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int first = span_of<VEC>(k * at.threads + at.lane, n).first;
    if (a.w) load_params<T>(a.w, a.wide, first, w[k]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (!a.w) w[k][e] = 1.0f;
      dw[k][e] = db[k][e] = 0.0f;
    }
  }
  int turn = 0;
  // One turn: the next one's rows are on their way while this one's are summed, if registers
  // hold both.
  auto step = [&](Row& r, Row& next) -> bool {
    const int64_t row = begin + at.group;
    const bool live = row < a.M, more = begin + stride < a.M;
    if (!AHEAD) fetch(r, row);
    V extra[SUM ? K : 1];
    if (SUM && live) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        extra[k] = load_vec((const T*)a.dsum + row * a.ldsum + span_of<VEC>(k * at.threads + at.lane, n).first);
    }
    if (AHEAD && more) fetch(next, row + stride);
    float s[2] = {0.0f, 0.0f};   // of g = dy w and of g c, c = h - mean
    if (live) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const Span span = span_of<VEC>(k * at.threads + at.lane, n);
        float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = (float)r.dy[k][e], c = (float)r.h[k][e] - r.mean, g = d * w[k][e];
          dw[k][e] += d * (c * r.rstd);
          db[k][e] += d;
          t1 += RAGGED && e < span.twice ? 0.0f : g;
          t2 += RAGGED && e < span.twice ? 0.0f : g * c;
        }
        s[0] += !RAGGED && span.twice ? 0.0f : t1;
        s[1] += !RAGGED && span.twice ? 0.0f : t2;
      }
    }
    row_sums<SUB>(s, at, meet[turn]);
    // dx = rstd (g - mean(g) - xhat mean(g xhat)) with xhat = c rstd
    const float shift = s[0] * inv_n * r.rstd, slope = s[1] * inv_n * r.rstd * r.rstd;
    if (live && a.dx) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const Span span = span_of<VEC>(k * at.threads + at.lane, n);
        if (span.twice == VEC) continue;
        V out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float c = (float)r.h[k][e] - r.mean;
          float d = (float)r.dy[k][e] * w[k][e] * r.rstd - shift;
          d -= c * r.rstd * slope;
          if (SUM) d += (float)extra[k][e];
          out[e] = (T)d;
        }
        store_vec((T*)a.dx + row * a.N + span.first, out);
      }
    }
    begin += stride;
    turn ^= 1;
    return more;
  };
  if (AHEAD) {
    while (step(one, other) && step(other, one)) {
    }
  } else {
    while (step(one, one)) {
    }
  }
  if (!a.partial) return;
  float* sums = a.partial + (int64_t)blockIdx.x * 2 * n;
  if (rows == 1) {   // (of elements that two vectors have, both have the same sums)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Span span = span_of<VEC>(k * at.threads + at.lane, n);
      if (span.twice == VEC) continue;
#pragma unroll
      for (int e = 0; e < VEC; e += 4) {
        store_vec(sums + span.first + e, Vec<float>::Type{dw[k][e], dw[k][e + 1], dw[k][e + 2], dw[k][e + 3]});
        store_vec(sums + n + span.first + e, Vec<float>::Type{db[k][e], db[k][e + 1], db[k][e + 2], db[k][e + 3]});
      }
    }
    return;
  }
  const int width = K * at.threads * VEC;   // of a row, vectors behind its end included
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float* mine = joined + at.group * 2 * width + (k * at.threads + at.lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      *(float4*)(mine + e) = float4{dw[k][e], dw[k][e + 1], dw[k][e + 2], dw[k][e + 3]};
      *(float4*)(mine + width + e) = float4{db[k][e], db[k][e + 1], db[k][e + 2], db[k][e + 3]};
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * width; c += blockDim.x) {
    const int place = c < width ? c : c - width;
    const Span span = span_of<VEC>(place / VEC, n);
    if (place % VEC < span.twice) continue;
    float s = 0.0f;
    for (int r = 0; r < rows; ++r) s += joined[r * 2 * width + c];
    sums[(c < width ? 0 : n) + span.first + place % VEC] = s;
  }
}

// The workgroups' sums added up: 32 of the 2 N columns to a workgroup, 16 threads to a column,
// each taking every 16th part: all loads of the launch are on their way at once, lines of 128 bytes
// each.  8 MB in 4 us; 16 columns to a workgroup 5.5, four columns to a thread 6.
constexpr int JOIN_COLUMNS = 32, JOIN_SLICES = 16;
template <typename T>
__global__ void __launch_bounds__(JOIN_COLUMNS* JOIN_SLICES) norm_grad_join_kernel(const NormGradArgs a) {
  __shared__ float shared[JOIN_SLICES][JOIN_COLUMNS];
  const int slice = threadIdx.x / JOIN_COLUMNS, lane = threadIdx.x % JOIN_COLUMNS;
  const int64_t all = 2 * a.N, col = block_number() * JOIN_COLUMNS + lane;
  float s = 0.0f;
  if (col < all) {
    const float* p = a.partial + col;
#pragma unroll 16
    for (int part = slice; part < a.parts; part += JOIN_SLICES) s += p[(int64_t)part * all];
  }
  shared[slice][lane] = s;
  __syncthreads();
  if (slice != 0 || col >= all) return;
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < JOIN_SLICES; ++i) total += shared[i][lane];
  void* out = col < a.N ? a.dw : a.db;
  const int64_t i = col < a.N ? col : col - a.N;
  if (!out) return;
  if (a.wide) ((float*)out)[i] = total; else ((T*)out)[i] = (T)total;
}

template <typename T>
int norm_grad_join(const NormGradArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(norm_grad_join_kernel<T>, grid_of(ceil_div(2 * a.N, JOIN_COLUMNS)), dim3(JOIN_COLUMNS * JOIN_SLICES), 0,
                     stream, a);
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

template <typename T, int K, bool SUB>
int norm_grad_rows_launch(NormGradArgs a, const RowPlan& plan, hipStream_t stream) {
  const bool params = a.dw || a.db;
  // as many rows at a time as 1024 threads hold, but all workgroups first
  const int fit = SUB ? 64 : 16 / plan.waves;
  const int64_t want = ceil_div(a.M, MOST_PARTS);
  int rows = want < fit ? (int)want : fit;
  if (SUB) rows = (rows + 3) / 4 * 4;   // (whole waves)
  const int threads = SUB ? rows * 16 : plan.waves * rows * 64;
  const int64_t groups = ceil_div(a.M, rows);
  a.parts = groups < MOST_PARTS ? (int)groups : MOST_PARTS;
  const size_t lds = params && rows > 1 ? (size_t)threads * 2 * K * Vec<T>::N * sizeof(float) : 0;
  constexpr size_t MOST_LDS = 1024 * 2 * K * Vec<T>::N * sizeof(float);
#define AXN_NORM_GRAD(RAGGED, SUM)                                                                                  \
  do {                                                                                                              \
    static std::atomic<unsigned long long> allowed{0};                                                              \
    if (lds > 32768) {                                                                                              \
      const int rc = allow_lds((const void*)norm_grad_rows_kernel<T, K, SUB, RAGGED, SUM>, MOST_LDS, allowed);      \
      if (rc) return rc;                                                                                            \
    }                                                                                                               \
    hipLaunchKernelGGL((norm_grad_rows_kernel<T, K, SUB, RAGGED, SUM>), dim3(a.parts), dim3(threads), lds, stream,  \
                       a, plan.waves, rows);                                                                        \
  } while (0)
  const bool ragged = a.N % Vec<T>::N != 0;
  if (ragged && a.dsum) AXN_NORM_GRAD(true, true);
  if (ragged && !a.dsum) AXN_NORM_GRAD(true, false);
  if (!ragged && a.dsum) AXN_NORM_GRAD(false, true);
  if (!ragged && !a.dsum) AXN_NORM_GRAD(false, false);
#undef AXN_NORM_GRAD
  AXN_HIP_TRY(hipGetLastError());
  return params ? norm_grad_join<T>(a, stream) : AXN_OK;
}

template <typename T>
int norm_grad_rows(const NormGradArgs& a, hipStream_t stream) {
  const RowPlan plan = plan_row(a.N, Vec<T>::N, true);
  if (plan.sub)
    return plan.k == 1 ? norm_grad_rows_launch<T, 1, true>(a, plan, stream) : norm_grad_rows_launch<T, 2, true>(a, plan, stream);
  if (plan.k == 1) return norm_grad_rows_launch<T, 1, false>(a, plan, stream);
  if (plan.k == 2) return norm_grad_rows_launch<T, 2, false>(a, plan, stream);
  return norm_grad_rows_launch<T, 4, false>(a, plan, stream);
}

// ------------------------------------------------------------- long rows ----
// Rows beyond the registers of 16 waves: a workgroup of them to a row, which it reads once for each
// sum and once more for the result, again from the caches.  Element by element with 256 threads
// 4 x 40000 bf16 took 101 us, so 10; 1000 x 100000 654, so 117 (3.4 TB/s), its backward 890 and 286.
constexpr int LONG_THREADS = 1024;

// The sum over a workgroup, in all of its threads.
template <int THREADS>
__device__ __forceinline__ float block_sum(float x, float* shared) {
  constexpr int WAVES = THREADS / 64;
  x = wave64_sum(x);
  __syncthreads();   // (the sums of an earlier call have been read)
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) x += shared[w];
  return x;
}

template <typename T>
__global__ void __launch_bounds__(LONG_THREADS) norm_long_kernel(const NormArgs a) {
  constexpr int VEC = Vec<T>::N;
  typedef typename Vec<T>::Type V;
  __shared__ float shared[LONG_THREADS / 64];
  const int64_t row = block_number();
  if (row >= a.M) return;
  const T *x = (const T*)a.x + row * a.ldx, *r = a.r ? (const T*)a.r + row * a.ldr : nullptr;
  const int n = (int)a.N, vectors = (n - 1) / VEC + 1;
  auto at = [&](int first) -> V {
    V v = load_vec(x + first);
    if (r) {
      const V o = load_vec(r + first);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = (T)((float)v[e] + (float)o[e]);
    }
    return v;
  };
  float s = 0.0f;
#pragma unroll 4
  for (int v = threadIdx.x; v < vectors; v += LONG_THREADS) {
    const Span span = long_span<VEC>(v, n);
    const V h = at(span.first);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += e < span.twice ? 0.0f : (float)h[e];
  }
  const float mean = block_sum<LONG_THREADS>(s, shared) / (float)n;
  s = 0.0f;
#pragma unroll 4
  for (int v = threadIdx.x; v < vectors; v += LONG_THREADS) {
    const Span span = long_span<VEC>(v, n);
    const V h = at(span.first);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = e < span.twice ? 0.0f : (float)h[e] - mean;
      s += d * d;
    }
  }
  const float rstd = 1.0f / sqrtf(block_sum<LONG_THREADS>(s, shared) / (float)n + a.eps);
  for (int v = threadIdx.x; v < vectors; v += LONG_THREADS) {
    const Span span = long_span<VEC>(v, n);
    const V h = at(span.first);
    float w[VEC], b[VEC];
    if (a.w) load_params<T>(a.w, a.wide, span.first, w);
    if (a.b) load_params<T>(a.b, a.wide, span.first, b);
    V y;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float f = ((float)h[e] - mean) * rstd * (a.w ? w[e] : 1.0f) + (a.b ? b[e] : 0.0f);
      asm volatile("" : "+v"(f));   // (see norm_rows_kernel)
      y[e] = (T)f;
    }
    store_vec((T*)a.y + row * a.N + span.first, y);
    if (r) store_vec((T*)a.h + row * a.N + span.first, h);
  }
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// dx of one row by a workgroup of THREADS, in vectors and from the caches the second time.
template <typename T, int THREADS>
__device__ __forceinline__ void dx_of_row(const NormGradArgs& a, int64_t row, float* shared) {
  constexpr int VEC = Vec<T>::N;
  typedef typename Vec<T>::Type V;
  const int n = (int)a.N, vectors = (n - 1) / VEC + 1;
  const T *dy = (const T*)a.dy + row * a.lddy, *h = (const T*)a.h + row * a.ldh;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float s1 = 0.0f, s2 = 0.0f, w[VEC];
#pragma unroll 2
  for (int v = threadIdx.x; v < vectors; v += THREADS) {
    const Span span = long_span<VEC>(v, n);
    const V d = load_vec(dy + span.first), x = load_vec(h + span.first);
    if (a.w) load_params<T>(a.w, a.wide, span.first, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float g = e < span.twice ? 0.0f : (float)d[e] * (a.w ? w[e] : 1.0f);
      s1 += g;
      s2 += e < span.twice ? 0.0f : g * ((float)x[e] - mean);
    }
  }
  const float shift = block_sum<THREADS>(s1, shared) / (float)n * rstd;
  const float slope = block_sum<THREADS>(s2, shared) / (float)n * rstd * rstd;
#pragma unroll 2
  for (int v = threadIdx.x; v < vectors; v += THREADS) {
    const Span span = long_span<VEC>(v, n);
    const V d = load_vec(dy + span.first), x = load_vec(h + span.first);
    V extra, out;
    if (a.dsum) extra = load_vec((const T*)a.dsum + row * a.ldsum + span.first);
    if (a.w) load_params<T>(a.w, a.wide, span.first, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float g = (float)d[e] * (a.w ? w[e] : 1.0f) * rstd - shift;
      g -= ((float)x[e] - mean) * rstd * slope;
      if (a.dsum) g += (float)extra[e];
      out[e] = (T)g;
    }
    store_vec((T*)a.dx + row * a.N + span.first, out);
  }
}

// Backward of few rows in one launch and without a workspace: the sums over rows need nothing of the
// sums along them.  The first a.M workgroups take a row each, in vectors and from the caches the
// second time, the others FEW_COLUMNS columns each and all rows, FEW_SLICES threads to a column.
constexpr int FEW_COLUMNS = 32, FEW_SLICES = 8, FEW_THREADS = FEW_COLUMNS * FEW_SLICES;
template <typename T>
__global__ void __launch_bounds__(FEW_THREADS) norm_grad_few_kernel(const NormGradArgs a) {
  __shared__ float shared[2][FEW_SLICES][FEW_COLUMNS];
  const int n = (int)a.N, rows = a.dx ? (int)a.M : 0, t = threadIdx.x;
  if ((int)blockIdx.x < rows) {
    dx_of_row<T, FEW_THREADS>(a, blockIdx.x, &shared[0][0][0]);
    return;
  }
  const int lane = t % FEW_COLUMNS, slice = t / FEW_COLUMNS;
  const int64_t col = (int64_t)(blockIdx.x - rows) * FEW_COLUMNS + lane;
  float dw = 0.0f, db = 0.0f;
  if (col < n) {
#pragma unroll 8
    for (int row = slice; row < (int)a.M; row += FEW_SLICES) {
      const float d = (float)((const T*)a.dy)[row * a.lddy + col];
      dw += d * (((float)((const T*)a.h)[row * a.ldh + col] - a.mean[row]) * a.rstd[row]);
      db += d;
    }
  }
  shared[0][slice][lane] = dw;
  shared[1][slice][lane] = db;
  __syncthreads();
  if (slice > 1 || col >= n) return;
  void* out = slice == 0 ? a.dw : a.db;
  if (!out) return;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < FEW_SLICES; ++i) s += shared[slice][i][lane];
  if (a.wide) ((float*)out)[col] = s; else ((T*)out)[col] = (T)s;
}

// Up to 512 rows (of 16 elements on, so that a vector fits, and up to 2^20, so that the grid does).  us, two
// launches / this one: 64 x 1024 fp32 7.4 / 5.0, 400 x 1024 10.1 / 6.0, 800 x 1024 10.6 / 11.3; 256 x 4096 bf16 10.6 / 5.5, 800 x 4096
// 14.7 / 12.5, 1100 x 4096 16.4 / 15.8; 128 x 12288 16.4 / 10.2, 600 x 12288 21.4 / 19.7, 800 x 12288 23.9 /
// 27.0; 400 x 8192 fp32 14.7 / 13.8, 600 x 8192 17.1 / 20.3.  At the rule's border, 513 rows in two launches
// / 512 in this one: bf16 x 1024 10.2 / 5.7, x 8192 16.7 / 10.5, x 16384 24.0 / 23.1, x 65536 89 / 88, x 2^20
// 1823 / 1699; fp32 x 1024 9.7 / 6.0, x 8192 16.5 / 16.9, x 16384 27.6 / 33.3, x 65536 174 / 137, x 2^20 3555
// / 2855.  So the rule loses on fp32 rows of some 8192 to 16384 elements, from 450 and 400 rows on.
inline bool few_rows(int64_t M, int64_t N) { return M >= 1 && M <= 512 && N >= 16 && N <= 1 << 20; }

template <typename T>
__global__ void __launch_bounds__(LONG_THREADS) norm_dx_long_kernel(const NormGradArgs a) {
  __shared__ float shared[LONG_THREADS / 64];
  const int64_t row = block_number();
  if (row < a.M) dx_of_row<T, LONG_THREADS>(a, row, shared);
}

// Column sums over the rows of one part: a thread to the columns of a vector.
template <typename T>
__global__ void __launch_bounds__(256) norm_dparam_long_kernel(const NormGradArgs a) {
  constexpr int VEC = Vec<T>::N;
  typedef typename Vec<T>::Type V;
  const int n = (int)a.N, v = blockIdx.x * 256 + threadIdx.x;
  if (v >= (n - 1) / VEC + 1) return;
  const int first_col = long_span<VEC>(v, n).first;   // (of columns that two have, both have the same sums)
  const int part = blockIdx.z;
  const int64_t first = a.M * part / a.parts, last = a.M * (part + 1) / a.parts;
  float dw[VEC], db[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) dw[e] = db[e] = 0.0f;
#pragma unroll 4
  for (int64_t row = first; row < last; ++row) {
    const V d = load_vec((const T*)a.dy + row * a.lddy + first_col), x = load_vec((const T*)a.h + row * a.ldh + first_col);
    const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      dw[e] += (float)d[e] * (((float)x[e] - mean) * rstd);
      db[e] += (float)d[e];
    }
  }
  float* sums = a.partial + (int64_t)part * 2 * n + first_col;
#pragma unroll
  for (int e = 0; e < VEC; e += 4) {
    store_vec(sums + e, Vec<float>::Type{dw[e], dw[e + 1], dw[e + 2], dw[e + 3]});
    store_vec(sums + n + e, Vec<float>::Type{db[e], db[e + 1], db[e + 2], db[e + 3]});
  }
}

// ------------------------------------------------------ rows below a vector --
// Rows of fewer elements than a vector has: a thread to a row.  1000000 x 4 bf16 forward 934 us with a
// workgroup to a row, 10 so; backward 1184 and 27.
template <typename T>
__global__ void __launch_bounds__(256) norm_tiny_kernel(const NormArgs a) {
  constexpr int MOST = Vec<T>::N - 1;
  const int n = (int)a.N;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.M; row += (int64_t)gridDim.x * 256) {
    float h[MOST], s = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      h[i] = 0.0f;
      if (i >= n) continue;
      h[i] = (float)((const T*)a.x)[row * a.ldx + i];
      if (a.r) {
        const T sum = (T)(h[i] + (float)((const T*)a.r)[row * a.ldr + i]);
        ((T*)a.h)[row * a.N + i] = sum;
        h[i] = (float)sum;
      }
      s += h[i];
    }
    const float mean = s / (float)n;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      h[i] -= mean;
      s += i < n ? h[i] * h[i] : 0.0f;
    }
    const float rstd = 1.0f / sqrtf(s / (float)n + a.eps);
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      if (i >= n) continue;
      float f = h[i] * rstd * (a.w ? param_at<T>(a.w, a.wide, i) : 1.0f) + (a.b ? param_at<T>(a.b, a.wide, i) : 0.0f);
      asm volatile("" : "+v"(f));   // (see norm_rows_kernel)
      ((T*)a.y)[row * a.N + i] = (T)f;
    }
    if (a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_grad_tiny_kernel(const NormGradArgs a) {
  constexpr int MOST = Vec<T>::N - 1;
  __shared__ float shared[4];
  const int n = (int)a.N;
  float dw[MOST], db[MOST], w[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    dw[i] = db[i] = 0.0f;
    w[i] = i < n && a.w ? param_at<T>(a.w, a.wide, i) : 1.0f;
  }
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.M; row += (int64_t)a.parts * 256) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[MOST], xhat[MOST], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      g[i] = xhat[i] = 0.0f;
      if (i >= n) continue;
      const float d = (float)((const T*)a.dy)[row * a.lddy + i];
      xhat[i] = ((float)((const T*)a.h)[row * a.ldh + i] - mean) * rstd;
      dw[i] += d * xhat[i];
      db[i] += d;
      g[i] = d * w[i];
      s1 += g[i];
      s2 += g[i] * xhat[i];
    }
    if (!a.dx) continue;
    s1 /= (float)n;
    s2 /= (float)n;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
      if (i >= n) continue;
      float d = (g[i] - s1 - xhat[i] * s2) * rstd;
      if (a.dsum) d += (float)((const T*)a.dsum)[row * a.ldsum + i];
      ((T*)a.dx)[row * a.N + i] = (T)d;
    }
  }
  if (!a.partial) return;
  float* sums = a.partial + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    if (i >= n) continue;   // (for all threads alike)
    const float sw = block_sum<256>(dw[i], shared), sb = block_sum<256>(db[i], shared);
    if (threadIdx.x == 0) {
      sums[i] = sw;
      sums[n + i] = sb;
    }
  }
}

// Into how many parts the rows are cut for the column sums of long ones: no more sums than rows to add,
// and fewer for wide ones, whose columns fill the GPU by themselves.
int norm_grad_parts(int64_t M, int64_t N) {
  int64_t parts = ceil_div(M, 16);
  if (parts > MOST_PARTS) parts = MOST_PARTS;
  const int64_t most = (1 << 25) / N;
  return (int)(parts <= most ? parts : most > 0 ? most : 1);
}

template <int DT>
int norm_launch(const NormArgs& a, hipStream_t stream) {
  typedef typename Elem<DT>::type T;
  if (a.N >= Vec<T>::N && a.N <= 4096 * Vec<T>::N) return norm_rows<T>(a, stream);
  if (a.N < Vec<T>::N) {
    const int64_t groups = ceil_div(a.M, 256);
    hipLaunchKernelGGL(norm_tiny_kernel<T>, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL(norm_long_kernel<T>, grid_of(a.M), dim3(LONG_THREADS), 0, stream, a);
  }
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

template <int DT>
int norm_grad_launch(NormGradArgs a, hipStream_t stream) {
  typedef typename Elem<DT>::type T;
  const bool params = a.dw || a.db;
  if (a.M == 0) return norm_grad_join<T>(a, stream);   // (sums of nothing)
  if (few_rows(a.M, a.N)) {
    const int64_t groups = (a.dx ? a.M : 0) + (params ? ceil_div(a.N, FEW_COLUMNS) : 0);
    hipLaunchKernelGGL(norm_grad_few_kernel<T>, dim3((unsigned)groups), dim3(FEW_THREADS), 0, stream, a);
    AXN_HIP_TRY(hipGetLastError());
    return AXN_OK;
  }
  if (!params) a.partial = nullptr;
  if (a.N >= Vec<T>::N && a.N <= 4096 * Vec<T>::N) return norm_grad_rows<T>(a, stream);
  if (a.N < Vec<T>::N) {
    const int64_t groups = ceil_div(a.M, 256);
    a.parts = groups < MOST_PARTS ? (int)groups : MOST_PARTS;
    hipLaunchKernelGGL(norm_grad_tiny_kernel<T>, dim3(a.parts), dim3(256), 0, stream, a);
    AXN_HIP_TRY(hipGetLastError());
    return params ? norm_grad_join<T>(a, stream) : AXN_OK;
  }
  if (a.dx) {
    hipLaunchKernelGGL(norm_dx_long_kernel<T>, grid_of(a.M), dim3(LONG_THREADS), 0, stream, a);
    AXN_HIP_TRY(hipGetLastError());
  }
  if (!params) return AXN_OK;
  a.parts = norm_grad_parts(a.M, a.N);
  const dim3 grid((unsigned)ceil_div(ceil_div(a.N, Vec<T>::N), 256), 1, a.parts);
  hipLaunchKernelGGL(norm_dparam_long_kernel<T>, grid, dim3(256), 0, stream, a);
  AXN_HIP_TRY(hipGetLastError());
  return norm_grad_join<T>(a, stream);
}

}  // namespace

size_t layer_norm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M < 1 || N < 1 || few_rows(M, N)) return 0;
  // (rows of up to 4096 vectors of 8: a sum of every workgroup, see norm_grad_rows_launch)
  const int64_t parts = N > 32768 ? norm_grad_parts(M, N) : M < MOST_PARTS ? M : MOST_PARTS;
  return (size_t)parts * 2 * (size_t)N * sizeof(float);
}

int launch_layer_norm_fwd(const void* x, const void* r, const void* w, const void* b, void* y, void* h, float* mean,
                          float* rstd, int dtype, bool wide, int64_t M, int64_t N, int64_t ldx, int64_t ldr, float eps,
                          hipStream_t stream) {
  const NormArgs a = {x, r, w, b, y, h, mean, rstd, M, N, ldx, ldr, eps, wide,
                      M * N * (dtype == AXN_F32 ? 4 : 2) <= kL2};
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
                          0, wide};
  switch (dtype) {
    case AXN_BF16: return norm_grad_launch<AXN_BF16>(a, stream);
    case AXN_F16: return norm_grad_launch<AXN_F16>(a, stream);
    default: return norm_grad_launch<AXN_F32>(a, stream);
  }
}

}  // namespace axn
