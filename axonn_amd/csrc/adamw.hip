// AdamW over a list of tensors (gfx950): Adam with the weight decay applied to the weights
// themselves, p <- (1 - lr decay) p - lr / bc1 m / (sqrt(v / bc2) + eps), in one pass that
// also unscales and clips the gradient and writes the low-precision copy of the weights.
//
//   mt_adamw    moments in fp32: the update of multi_tensor.h with this arithmetic
//   mt_adamw8   moments in 8 bits, 256 elements to a block
//   adamw8_moments   8-bit moments as numbers
//
// 8-bit moments.  A block has one exponent byte E for each moment: the exponent field of its
// largest magnitude as a float, the next one from a mantissa of 1.875 on; 255 marks a block
// that is not finite.  A code of the first moment is a sign, 4 bits of exponent and 3 of
// mantissa, one of the second moment 5 and 3, both with gradual underflow:
//   F(c) = c / 8  (c < 8),  (1 + (c & 7) / 8) 2^((c >> 3) - 1)  otherwise,
//   m = +-F(c) 2^(E - 141),  v = F(c) 2^(E - 157),
// so that the largest magnitude lies in the codes' top octave and powers of two are all that a
// value is scaled by: c << 20 are the bits of F(c) 2^-126, a float may be denormal, and both
// directions are one ldexp.
// Rounding is stochastic: a value between two codes takes the upper one with the probability
// of its place between them.  Rounded to nearest, second moments would stand still: a step
// changes one by (1 - beta2) (g^2 - v), some thousandth of it, a code by a sixteenth to an
// eighth of it.  A second moment that is not zero keeps at least code 1, so that a first
// moment that is still there is not divided by eps alone.
// The moments' arithmetic rounds each product and each sum by itself, and E, the codes' places
// and the random words are integer work: codes are the same on every machine that follows the
// formulas.
#include "axn_internal.h"
#include "multi_tensor.h"

namespace axn {
namespace {

struct AdamWScalars {
  axn_adamw_hparams hp;
  float inv_scale;
};

__device__ __forceinline__ void adamw_math(float g, float& p, float& m, float& v, const AdamWScalars& s, float gmul) {
  g = g * s.inv_scale;
  g = g * gmul;
  m = m + (g - m) * s.hp.one_minus_beta1;
  v = v * s.hp.beta2 + s.hp.one_minus_beta2 * g * g;
  const float denom = sqrtf(v) * s.hp.inv_sqrt_bc2 + s.hp.eps;
  p = p * s.hp.keep - s.hp.lr_over_bc1 * (m / denom);
  // (the low-precision copy is the rounding of the fp32 value that is stored, see adam_math)
  asm volatile("" : "+v"(p));
}

template <int GDT, int PDT, bool HAS_PLOW, bool HAS_SCAN>
__global__ void __launch_bounds__(ADAM_THREADS)
    mt_adamw_kernel(const MtTable tab, const AdamWScalars s, const axn_scan_result* scan) {
  const int b = blockIdx.x;
  const TensorRow row = row_by_scalar_search(tab, b);
  int found_inf = 0;
  float gmul = 1.0f;
  if (HAS_SCAN) {   // (beside the lookup, not in front of it)
    found_inf = scan->found_inf;
    gmul = scan->clip_coef;
  }
  update_chunk<GDT, PDT, HAS_PLOW>(row, b, found_inf, gmul, [&](float g, float& p, float& m, float& v, float mul) {
    adamw_math(g, p, m, v, s, mul);
  });
}

// ------------------------------------------------------------- 8-bit codes --
constexpr int BLOCK8 = 256;             // elements of a block
constexpr int M_BIAS = 15, V_BIAS = 31; // value = ldexp(float with bits c << 20, E - bias)
constexpr int NOT_FINITE = 255;
constexpr int64_t kMostBlocks8 = (1 << 26) - 1;   // of a launch: below 2^32 threads

__device__ __forceinline__ float decode_m(uint32_t c, int e) {
  return ldexpf(__uint_as_float((c & 0x7fu) << 20 | (c & 0x80u) << 24), e - M_BIAS);
}
__device__ __forceinline__ float decode_v(uint32_t c, int e) {
  return ldexpf(__uint_as_float(c << 20), e - V_BIAS);
}
// E of a block whose largest magnitude has these bits (of a NaN: 255 too).
__device__ __forceinline__ int exponent_of(uint32_t bits) {
  const uint32_t e = (bits + 0x100000u) >> 23;
  return e > NOT_FINITE ? NOT_FINITE : (int)e;
}
// The code of a magnitude of at most E's, `word`'s 16 bits being the place from which on the
// upper one of its two neighbours is taken.
__device__ __forceinline__ uint32_t encode(float magnitude, int e, int bias, uint32_t word) {
  return (__float_as_uint(ldexpf(magnitude, bias - e)) + (word << 4 | 8u)) >> 20;
}

// The random words of the four elements q * 4 ... of the list: a counter, two keys, two
// rounds of multiplying and folding (odd constants from the golden ratio and the square roots
// of 2, 3, 11, 17 and 19).  The low half is the first moment's, the high one the second's.
__device__ __forceinline__ void random_words(uint64_t q, uint32_t k0, uint32_t k1, uint32_t (&w)[4]) {
  uint32_t x = ((uint32_t)q ^ k0) * 0x9E3779B9u;
  x = ((x ^ x >> 16) + k1 + (uint32_t)(q >> 32)) * 0x6A09E667u;
  x ^= x >> 15;
  const uint32_t c[4] = {0xBB67AE85u, 0x510E527Fu, 0x1F83D9ABu, 0x5BE0CD19u};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = x * c[e];
    w[e] ^= w[e] >> 16;
  }
}

struct AdamW8Scalars {
  AdamWScalars s;
  uint32_t k0, k1;        // the seed's halves
  int64_t first_block;    // number of the launch's first block in the list
};

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, o, 64);
    x = y > x ? y : x;
  }
  return x;
}

// One block of 256 elements a wave, four to a lane, element by element.
template <int GDT, int PDT, bool HAS_PLOW, bool HAS_SCAN>
__global__ void __launch_bounds__(64)
    mt_adamw8_kernel(const MtTable tab, const AdamW8Scalars a, const axn_scan_result* scan) {
  typedef typename Lowp<GDT>::raw graw;
  typedef typename Lowp<PDT>::raw praw;
  const int b = blockIdx.x, lane = threadIdx.x;
  const TensorRow row = row_by_scalar_search(tab, b);
  float gmul = 1.0f;
  if (HAS_SCAN) {
    if (scan->found_inf != 0) return;   // the whole step is skipped
    gmul = scan->clip_coef;
  }
  const int64_t block = b - row.first_chunk;
  const int64_t first = block * BLOCK8 + lane * 4;
  const int64_t left = row.size - first;
  const int count = left >= 4 ? 4 : left > 0 ? (int)left : 0;
  uint32_t* codes = (uint32_t*)row.m + block * (2 * BLOCK8 / 4) + lane * 2;
  uint8_t* exps = (uint8_t*)row.v + block * 2;
  const uint32_t cm = codes[0], cv = codes[1];
  const int em = exps[0], ev = exps[1];
  float m[4], v[4];
  uint32_t largest_m = 0, largest_v = 0;
  for (int e = 0; e < 4; ++e) {
    m[e] = em == NOT_FINITE ? __builtin_nanf("") : decode_m(cm >> (8 * e) & 0xffu, em);
    v[e] = ev == NOT_FINITE ? __builtin_nanf("") : decode_v(cv >> (8 * e) & 0xffu, ev);
    if (e >= count) m[e] = v[e] = 0.0f;   // (behind the tensor's end)
    if (e < count) {
#pragma clang fp contract(off)
      float g = Lowp<GDT>::to_float(((const graw*)row.g)[first + e]) * a.s.inv_scale;
      g = g * gmul;
      const float step_m = (g - m[e]) * a.s.hp.one_minus_beta1;
      m[e] = m[e] + step_m;
      const float square = a.s.hp.one_minus_beta2 * g * g;
      v[e] = v[e] * a.s.hp.beta2 + square;
      float p = row.p[first + e];
      const float denom = sqrtf(v[e]) * a.s.hp.inv_sqrt_bc2 + a.s.hp.eps;
      p = p * a.s.hp.keep - a.s.hp.lr_over_bc1 * (m[e] / denom);
      row.p[first + e] = p;
      if (HAS_PLOW) ((praw*)row.plow)[first + e] = Lowp<PDT>::from_float(p);
    }
    const uint32_t bm = __float_as_uint(m[e]) & 0x7fffffffu, bv = __float_as_uint(v[e]) & 0x7fffffffu;
    largest_m = bm > largest_m ? bm : largest_m;
    largest_v = bv > largest_v ? bv : largest_v;
  }
  const int nm = exponent_of(wave_max(largest_m)), nv = exponent_of(wave_max(largest_v));
  uint32_t words[4], out_m = 0, out_v = 0;
  random_words((uint64_t)(a.first_block + b) * 64 + lane, a.k0, a.k1, words);
  for (int e = 0; e < 4; ++e) {
    uint32_t c = nm == NOT_FINITE ? 0u : encode(fabsf(m[e]), nm, M_BIAS, words[e] & 0xffffu);
    out_m |= (c | (m[e] < 0.0f ? 0x80u : 0u)) << (8 * e);
    c = nv == NOT_FINITE ? 0u : encode(v[e], nv, V_BIAS, words[e] >> 16);
    if (c == 0 && v[e] > 0.0f) c = 1;
    out_v |= c << (8 * e);
  }
  codes[0] = out_m;
  codes[1] = out_v;
  if (lane == 0) {
    exps[0] = (uint8_t)nm;
    exps[1] = (uint8_t)nv;
  }
}

template <int DT>
__global__ void __launch_bounds__(256)
    adamw8_moments_kernel(const uint32_t* codes, const uint8_t* exps, void* m, void* v, int64_t n) {
  typedef typename Lowp<DT>::raw raw;
  const int64_t first = (block_number() * 256 + threadIdx.x) * 4;
  if (first >= n) return;
  const int64_t block = first / BLOCK8;
  const uint32_t cm = codes[first / 2], cv = codes[first / 2 + 1];
  const int em = exps[2 * block], ev = exps[2 * block + 1];
  for (int e = 0; e < 4 && first + e < n; ++e) {
    if (m) ((raw*)m)[first + e] = Lowp<DT>::from_float(em == NOT_FINITE ? __builtin_nanf("") : decode_m(cm >> (8 * e) & 0xffu, em));
    if (v) ((raw*)v)[first + e] = Lowp<DT>::from_float(ev == NOT_FINITE ? __builtin_nanf("") : decode_v(cv >> (8 * e) & 0xffu, ev));
  }
}

template <int GDT, bool HAS_SCAN>
int adamw_launch(const Group& gr, const AdamWScalars& s, int plow_dtype, bool has_plow, const axn_scan_result* scan,
                 hipStream_t stream) {
  const dim3 grid((unsigned)gr.blocks), block(ADAM_THREADS);
  if (!has_plow)
    hipLaunchKernelGGL((mt_adamw_kernel<GDT, AXN_BF16, false, HAS_SCAN>), grid, block, ADAM_LDS, stream, gr.tab, s, scan);
  else if (plow_dtype == AXN_BF16)
    hipLaunchKernelGGL((mt_adamw_kernel<GDT, AXN_BF16, true, HAS_SCAN>), grid, block, ADAM_LDS, stream, gr.tab, s, scan);
  else
    hipLaunchKernelGGL((mt_adamw_kernel<GDT, AXN_F16, true, HAS_SCAN>), grid, block, ADAM_LDS, stream, gr.tab, s, scan);
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

template <int GDT, bool HAS_SCAN>
int adamw8_launch(const Group& gr, const AdamW8Scalars& a, int plow_dtype, bool has_plow, const axn_scan_result* scan,
                  hipStream_t stream) {
  const dim3 grid((unsigned)gr.blocks), block(64);
  if (!has_plow)
    hipLaunchKernelGGL((mt_adamw8_kernel<GDT, AXN_BF16, false, HAS_SCAN>), grid, block, 0, stream, gr.tab, a, scan);
  else if (plow_dtype == AXN_BF16)
    hipLaunchKernelGGL((mt_adamw8_kernel<GDT, AXN_BF16, true, HAS_SCAN>), grid, block, 0, stream, gr.tab, a, scan);
  else
    hipLaunchKernelGGL((mt_adamw8_kernel<GDT, AXN_F16, true, HAS_SCAN>), grid, block, 0, stream, gr.tab, a, scan);
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

template <int GDT>
int adamw8_dispatch(const Group& gr, const AdamW8Scalars& a, int plow_dtype, bool has_plow, const axn_scan_result* scan,
                    hipStream_t stream) {
  return scan != nullptr ? adamw8_launch<GDT, true>(gr, a, plow_dtype, has_plow, scan, stream)
                         : adamw8_launch<GDT, false>(gr, a, plow_dtype, has_plow, scan, stream);
}

}  // namespace

int launch_mt_adamw(const void* const* h_g, void* const* h_p, void* const* h_m, void* const* h_v, void* const* h_plow,
                    const int64_t* h_sizes, int64_t n, int g_dtype, int plow_dtype, float inv_scale,
                    const axn_scan_result* scan, const axn_adamw_hparams& hp, hipStream_t stream) {
  const void* const* sets[5] = {h_g, (const void* const*)h_p, (const void* const*)h_m, (const void* const*)h_v,
                                (const void* const*)h_plow};
  const int es[5] = {dtype_size(g_dtype), 4, 4, 4, dtype_size(plow_dtype)};
  AdamWScalars s;
  s.hp = hp;
  s.inv_scale = inv_scale;
  const bool has_plow = h_plow != nullptr;
  return for_each_group(sets, es, 5, h_sizes, n, ADAM_CHUNK, [&](const Group& gr) {
    switch (g_dtype) {
#define AXN_ADAMW_CASE(GDT)                                                                    \
  return scan != nullptr ? adamw_launch<GDT, true>(gr, s, plow_dtype, has_plow, scan, stream)  \
                         : adamw_launch<GDT, false>(gr, s, plow_dtype, has_plow, scan, stream)
      case AXN_BF16: AXN_ADAMW_CASE(AXN_BF16);
      case AXN_F16: AXN_ADAMW_CASE(AXN_F16);
      default: AXN_ADAMW_CASE(AXN_F32);
#undef AXN_ADAMW_CASE
    }
  });
}

int launch_mt_adamw8(const void* const* h_g, void* const* h_p, void* const* h_codes, void* const* h_exponents,
                     void* const* h_plow, const int64_t* h_sizes, int64_t n, int g_dtype, int plow_dtype, float inv_scale,
                     uint64_t seed, const axn_scan_result* scan, const axn_adamw_hparams& hp, hipStream_t stream) {
  AdamW8Scalars a;
  a.s.hp = hp;
  a.s.inv_scale = inv_scale;
  a.k0 = (uint32_t)seed;
  a.k1 = (uint32_t)(seed >> 32);
  a.first_block = 0;
  Group cur;
  cur.tab = MtTable();
  cur.blocks = 0;
  int k = 0;
  auto flush = [&]() -> int {
    if (k == 0) return AXN_OK;
    cur.tab.n = k;
    cur.tab.chunk = BLOCK8;
    for (int j = k; j <= MT_MAX; ++j) cur.tab.chunk_start[j] = j == k ? cur.blocks : 0x7fffffff;
    int rc;
    switch (g_dtype) {
      case AXN_BF16: rc = adamw8_dispatch<AXN_BF16>(cur, a, plow_dtype, h_plow != nullptr, scan, stream); break;
      case AXN_F16: rc = adamw8_dispatch<AXN_F16>(cur, a, plow_dtype, h_plow != nullptr, scan, stream); break;
      default: rc = adamw8_dispatch<AXN_F32>(cur, a, plow_dtype, h_plow != nullptr, scan, stream); break;
    }
    a.first_block += cur.blocks;
    cur.tab = MtTable();
    cur.blocks = 0;
    k = 0;
    return rc;
  };
  for (int64_t i = 0; i < n; ++i) {
    if (h_sizes[i] == 0) continue;
    const int64_t blocks = (h_sizes[i] + BLOCK8 - 1) / BLOCK8;
    if (blocks > kMostBlocks8) {
      set_error("multi-tensor: tensor %lld has too many elements (%lld)", (long long)i, (long long)h_sizes[i]);
      return AXN_ELIMIT;
    }
    if (k == MT_MAX || (int64_t)cur.blocks + blocks > kMostBlocks8) {
      const int rc = flush();
      if (rc != AXN_OK) return rc;
    }
    cur.tab.g[k] = h_g[i];
    cur.tab.p[k] = h_p[i];
    cur.tab.m[k] = h_codes[i];
    cur.tab.v[k] = h_exponents[i];
    cur.tab.plow[k] = h_plow ? h_plow[i] : nullptr;
    cur.tab.size[k] = h_sizes[i];
    cur.tab.chunk_start[k] = cur.blocks;
    cur.blocks += (int)blocks;
    ++k;
  }
  return flush();
}

int launch_adamw8_moments(const void* codes, const void* exponents, void* m, void* v, int dtype, int64_t n,
                          hipStream_t stream) {
  const dim3 grid = grid_of((n + 1023) / 1024), block(256);
  if (dtype == AXN_BF16)
    hipLaunchKernelGGL(adamw8_moments_kernel<AXN_BF16>, grid, block, 0, stream, (const uint32_t*)codes,
                       (const uint8_t*)exponents, m, v, n);
  else
    hipLaunchKernelGGL(adamw8_moments_kernel<AXN_F32>, grid, block, 0, stream, (const uint32_t*)codes,
                       (const uint8_t*)exponents, m, v, n);
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

}  // namespace axn
