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
constexpr int LDS8 = 7168;   // LDS that a workgroup reserves and never touches, see mt_adamw8_kernel
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

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
  return y > x ? y : x;
}
// The wave's largest, a scalar: rotations within the rows of 16 lanes, then the rows' four.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = dpp_max<0x128>(x);
  x = dpp_max<0x124>(x);
  x = dpp_max<0x122>(x);
  x = dpp_max<0x121>(x);
  const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16),
                 c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}

// Four of a block's elements, in a lane.
struct Four {
  float m[4], v[4];
};

__device__ __forceinline__ Four decode4(u32x2 codes, int em, int ev) {
  Four x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x.m[e] = decode_m(codes[0] >> (8 * e) & 0xffu, em);
    x.v[e] = decode_v(codes[1] >> (8 * e) & 0xffu, ev);
  }
  if (em == NOT_FINITE) {   // (the wave's: a scalar branch)
#pragma unroll
    for (int e = 0; e < 4; ++e) x.m[e] = __builtin_nanf("");
  }
  if (ev == NOT_FINITE) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x.v[e] = __builtin_nanf("");
  }
  return x;
}

// One element's step.  The moments' products and sums are rounded one by one; the weight's are
// not, its quotient and root are the instructions' of 1 ulp: an update's last bits are far
// below the weight's.
__device__ __forceinline__ void adamw8_math(float g, float& p, float& m, float& v, const AdamWScalars& s, float gmul) {
#pragma clang fp contract(off)
  g = g * s.inv_scale;
  g = g * gmul;
  const float change = (g - m) * s.hp.one_minus_beta1;
  m = m + change;
  const float square = s.hp.one_minus_beta2 * g * g;
  v = v * s.hp.beta2 + square;
  {
#pragma clang fp contract(fast)
    // (the root of a number below 2^-96 by way of 2^64 times it)
    const bool small = v < 0x1p-96f;
    float root = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v);
    root = small ? root * 0x1p-32f : root;
    float denom = root * s.hp.inv_sqrt_bc2 + s.hp.eps;
    denom = denom < 0x1p-126f ? 0x1p-126f : denom;   // (its reciprocal stays finite; a NaN stays one)
    p = p * s.hp.keep - s.hp.lr_over_bc1 * (m * __builtin_amdgcn_rcpf(denom));
  }
  asm volatile("" : "+v"(p));   // (the copy is the rounding of the fp32 value that is stored)
}

__device__ __forceinline__ uint32_t max_bits(const float (&x)[4]) {
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
    largest = b > largest ? b : largest;
  }
  return largest;
}
// The top bytes of four words.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&x)[4]) {
  const uint32_t lo = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0703u), hi = __builtin_amdgcn_perm(x[3], x[2], 0x07030c0cu);
  return lo | hi;
}

__device__ __forceinline__ u32x2 encode4(const Four& x, int em, int ev, const uint32_t (&words)[4]) {
  uint32_t m[4], v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // (a magnitude of at most E's; the word's 16 bits are the place from which on the upper one of its two neighbours is
    // taken) a code's bits are 20 to 27 of the sum; 4 up they are the top byte, the sign above the code
    m[e] = (__float_as_uint(ldexpf(fabsf(x.m[e]), M_BIAS - em)) + (words[e] << 4 & 0xffff0u | 8u)) << 4;
    m[e] |= x.m[e] < 0.0f ? 0x80000000u : 0u;
    v[e] = (__float_as_uint(ldexpf(x.v[e], V_BIAS - ev)) + (words[e] >> 12 & 0xffff0u | 8u)) << 4;
    const uint32_t least = x.v[e] > 0.0f ? 1u << 24 : 0u;
    v[e] = v[e] > least ? v[e] : least;
  }
  u32x2 codes;
  codes[0] = em == NOT_FINITE ? 0u : top_bytes(m);
  codes[1] = ev == NOT_FINITE ? 0u : top_bytes(v);
  return codes;
}

// A wave takes a block, four elements in a lane.  Figures of 5e8 elements in 64 tensors, bf16
// gradients and copies: 1.25 ms, 6.4 of the 6.8 TB/s of a copy, by the update's rules (see
// update_chunk).  The waves in flight matter here too: with the 28 registers of a lane all 32 a CU
// holds are 5 % slower (6.1), 22 are the best found (LDS8; 18: 6.1, 32-bit gradients 6.5 with
// each); two or four blocks of a wave, loads in front, lose 1 and 4 %.  Arithmetic is some 65
// operations an element, two thirds of what the time has room for: a precise root and quotient
// would be 20 more.
template <int GDT, int PDT, bool HAS_PLOW, bool HAS_SCAN>
__global__ void __launch_bounds__(64)
    mt_adamw8_kernel(const MtTable tab, const AdamW8Scalars a, const axn_scan_result* scan) {
  typedef typename Lowp<GDT>::raw graw;
  typedef typename Lowp<PDT>::raw praw;
  constexpr int GSZ = (int)sizeof(graw), PSZ = (int)sizeof(praw);
  const int b = blockIdx.x, lane = threadIdx.x, e0 = lane * 4;
  const TensorRow row = row_by_scalar_search(tab, b);
  int found_inf = 0;
  float gmul = 1.0f;
  if (HAS_SCAN) {   // (beside the lookup, not in front of it)
    found_inf = scan->found_inf;
    gmul = scan->clip_coef;
  }
  const int64_t block = b - row.first_chunk, begin = block * BLOCK8;
  // elements of the tensor from the block's first on; none if the step is skipped
  int64_t left = found_inf != 0 ? 0 : row.size - begin;
  if (left > BLOCK8) left = BLOCK8;
  if (left <= 0) return;
  const int count = (int)left, whole = count / 4 * 4;
  const bool vector = (row.meta & 0x100) != 0;
  auto stream = [&](const void* base, int64_t offset, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + offset), 0, bytes, 0x00020000);
  };
  // Buffers of the block's whole vectors; the lanes behind them load zeros and store nothing.
  const int in_vectors = vector ? whole : 0;
  const __amdgpu_buffer_rsrc_t bg = stream(row.g, begin * GSZ, in_vectors * GSZ), bp = stream(row.p, begin * 4, in_vectors * 4),
                               bl = stream(HAS_PLOW ? row.plow : (void*)row.p, begin * PSZ, in_vectors * PSZ),
                               bc = stream(row.m, block * 2 * BLOCK8, 2 * BLOCK8), be = stream(row.v, block * 2, 2);
  float g[4];
  const uint32_t exps = __builtin_amdgcn_raw_buffer_load_b16(be, 0, 0, 0);
  const u32x2 codes = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(bc, e0 * 2, 0, ADAM_LOAD_POLICY));
  if (GSZ == 2) {
    const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(bg, e0 * 2, 0, ADAM_LOAD_POLICY));
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = Lowp<GDT>::to_float((graw)(w[e / 2] >> (16 * (e & 1))));
  } else {
    const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bg, e0 * 4, 0, ADAM_LOAD_POLICY));
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = Lowp<GDT>::to_float((graw)w[e]);
  }
  f32x4 p = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bp, e0 * 4, 0, ADAM_LOAD_POLICY));
  __builtin_amdgcn_sched_barrier(0);   // every load is issued before the arithmetic
  // elements one by one: of the last, short vector, or of a tensor that is not aligned
  const int singles = !vector || e0 == whole ? min(max(count - e0, 0), 4) : 0;
  if (singles > 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < singles) {
        g[e] = Lowp<GDT>::to_float(((const graw*)row.g)[begin + e0 + e]);
        p[e] = row.p[begin + e0 + e];
      }
  }
  Four x = decode4(codes, __builtin_amdgcn_readfirstlane(exps & 0xffu), __builtin_amdgcn_readfirstlane(exps >> 8));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float pe = p[e];
    adamw8_math(g[e], pe, x.m[e], x.v[e], a.s, gmul);
    p[e] = pe;
  }
  if (e0 + 4 > count) {   // (behind the tensor's end, of a block that is not finite too)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e0 + e >= count) x.m[e] = x.v[e] = 0.0f;
  }
  uint32_t words[4];
  random_words((uint64_t)(a.first_block + b) * 64 + lane, a.k0, a.k1, words);
  const int em = exponent_of(wave_max(max_bits(x.m))), ev = exponent_of(wave_max(max_bits(x.v)));
  const u32x2 out = encode4(x, em, ev, words);
  praw low[4];
  if (HAS_PLOW) {
#pragma unroll
    for (int e = 0; e < 4; ++e) low[e] = Lowp<PDT>::from_float(p[e]);
  }
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, p), bp, e0 * 4, 0, ADAM_STORE_POLICY);
  __builtin_amdgcn_raw_buffer_store_b64(out, bc, e0 * 2, 0, ADAM_STORE_POLICY);
  if (HAS_PLOW) {
    u32x2 w;
    w[0] = (uint32_t)low[0] | (uint32_t)low[1] << 16;
    w[1] = (uint32_t)low[2] | (uint32_t)low[3] << 16;
    __builtin_amdgcn_raw_buffer_store_b64(w, bl, e0 * 2, 0, ADAM_STORE_POLICY);
  }
  if (lane == 0) __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(em | ev << 8), be, 0, 0, 0);
  if (singles > 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < singles) {
        row.p[begin + e0 + e] = p[e];
        if (HAS_PLOW) ((praw*)row.plow)[begin + e0 + e] = low[e];
      }
  }
}

// Four elements to a lane, a block to a wave, stored as vectors where m and v allow it.  5e8
// elements as bf16: 0.49 ms, 6.1 TB/s (workgroups of four waves 0.51; codes that were written just
// before come from the cache: not loaded past it, which gains 3 % where they do not).
template <int DT>
__global__ void __launch_bounds__(64)
    adamw8_moments_kernel(const u32x2* codes, const uint16_t* exps, void* m, void* v, int64_t n, int vector) {
  typedef typename Lowp<DT>::raw raw;
  typedef raw raw4 __attribute__((ext_vector_type(4)));
  const int64_t four = block_number() * 64 + threadIdx.x, first = four * 4;
  if (first >= n) return;
  // (a wave's elements are a block's)
  const uint32_t e2 = __builtin_amdgcn_readfirstlane(exps[first / BLOCK8]);
  const Four x = decode4(codes[four], e2 & 0xffu, e2 >> 8);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    raw* out = (raw*)(which == 0 ? m : v) + first;
    if ((which == 0 ? m : v) == nullptr) continue;
    raw4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = Lowp<DT>::from_float(which == 0 ? x.m[e] : x.v[e]);
    if (vector && first + 4 <= n) {
      __builtin_nontemporal_store(w, (raw4*)out);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (first + e < n) out[e] = w[e];
    }
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
    hipLaunchKernelGGL((mt_adamw8_kernel<GDT, AXN_BF16, false, HAS_SCAN>), grid, block, LDS8, stream, gr.tab, a, scan);
  else if (plow_dtype == AXN_BF16)
    hipLaunchKernelGGL((mt_adamw8_kernel<GDT, AXN_BF16, true, HAS_SCAN>), grid, block, LDS8, stream, gr.tab, a, scan);
  else
    hipLaunchKernelGGL((mt_adamw8_kernel<GDT, AXN_F16, true, HAS_SCAN>), grid, block, LDS8, stream, gr.tab, a, scan);
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
  return for_each_group(sets, es, 5, h_sizes, n, ADAM_CHUNK, ADAM_THREADS, [&](const Group& gr) {
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
    const int64_t blocks = ceil_div(h_sizes[i], BLOCK8);
    if (blocks > kMostBlocks8) {
      set_error("multi-tensor: tensor %lld has too many elements (%lld)", (long long)i, (long long)h_sizes[i]);
      return AXN_ELIMIT;
    }
    if (k == MT_MAX || cur.blocks + blocks > kMostBlocks8) {
      const int rc = flush();
      if (rc != AXN_OK) return rc;
    }
    const bool vector = (uintptr_t)h_p[i] % 16 == 0 && (uintptr_t)h_g[i] % (g_dtype == AXN_F32 ? 16 : 8) == 0 &&
                        (h_plow == nullptr || (uintptr_t)h_plow[i] % 8 == 0);
    cur.tab.g[k] = h_g[i];
    cur.tab.p[k] = h_p[i];
    cur.tab.m[k] = h_codes[i];
    cur.tab.v[k] = h_exponents[i];
    cur.tab.plow[k] = h_plow ? h_plow[i] : nullptr;
    cur.tab.size[k] = h_sizes[i];
    cur.tab.chunk_start[k] = cur.blocks;
    cur.tab.meta[k] = vector ? 0x100 : 0;
    cur.blocks += (int)blocks;
    ++k;
  }
  return flush();
}

int launch_adamw8_moments(const void* codes, const void* exponents, void* m, void* v, int dtype, int64_t n,
                          hipStream_t stream) {
  const dim3 grid = grid_of(ceil_div(n, BLOCK8)), block(64);
  const int vector = ((uintptr_t)m | (uintptr_t)v) % (4 * dtype_size(dtype)) == 0;
  if (dtype == AXN_BF16)
    hipLaunchKernelGGL(adamw8_moments_kernel<AXN_BF16>, grid, block, 0, stream, (const u32x2*)codes,
                       (const uint16_t*)exponents, m, v, n, vector);
  else
    hipLaunchKernelGGL(adamw8_moments_kernel<AXN_F32>, grid, block, 0, stream, (const u32x2*)codes,
                       (const uint16_t*)exponents, m, v, n, vector);
  AXN_HIP_TRY(hipGetLastError());
  return AXN_OK;
}

}  // namespace axn
