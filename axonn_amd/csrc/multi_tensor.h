// What the multi-tensor kernels share: how the tensors of a list are addressed, and the
// update's way through memory (one read-modify-write pass over gradients, fp32 weights and
// moments), which the Adam kernels of optim.hip and adamw.hip run with their own arithmetic.
//
// Addressing.  The tensors of one launch (at most MT_MAX) travel in the kernel
// argument block: pointers, sizes and a prefix sum of per-tensor chunk counts.
// Workgroup b finds its tensor in that prefix sum with scalar loads from the argument
// block (binary search; the update kernel's two-step search is described there) and owns
// one chunk of consecutive elements of it.
// Tensors are views into flat buffers at arbitrary element offsets
// (axonn/utils.py:11-30), so each tensor starts with a scalar "head" of up to 63
// elements after which every pointer of the tensor is 16-byte aligned (and on a
// cache line when the buffers allow it); the body is then moved as 16-byte vectors
// (8-byte ones for 16-bit streams of the update kernel).  A
// tensor whose pointers cannot be aligned by one common head is processed with
// scalar accesses.
#pragma once
#include "axn_internal.h"

namespace axn {
namespace {

constexpr int MT_MAX = 64;         // tensors per launch
// The read-modify-write update does best with one-wave workgroups that make one trip of
// ADAM_VECS 4-element vectors per lane (see update_chunk).
constexpr int ADAM_VEC = 4;                     // elements per vector of the update kernel
constexpr int ADAM_THREADS = 64;                // lanes per workgroup of the update kernel
constexpr int ADAM_VECS = 1;                    // vectors per lane
constexpr int ADAM_CHUNK = ADAM_THREADS * ADAM_VEC * ADAM_VECS;
// LDS the update kernel reserves per workgroup and never touches: it bounds the
// workgroups that are resident on a CU (160 KB per CU), see update_chunk.
constexpr int ADAM_LDS = 15360;
// Cache policy bits of the update kernel's buffer accesses (1 sc0, 2 nt, 16 sc1).  Loads
// non-temporal; stores non-temporal and written through (nt + sc1): 1 to 2 % over nt
// alone, 10 % over plain stores, measured on MI355X.
constexpr int ADAM_LOAD_POLICY = 2, ADAM_STORE_POLICY = 2 | 16;
static_assert(ADAM_THREADS >= 64 && ADAM_THREADS % 64 == 0, "a tensor's scalar head (up to 63 elements) is one element per lane");
static_assert(ADAM_CHUNK % 8 == 0, "chunks keep the 16-byte alignment of the tensor's body");
static_assert(ADAM_LDS <= 65536, "dynamic LDS a launch may ask for without a function attribute");

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

struct MtTable {
  const void* g[MT_MAX];
  void* p[MT_MAX];
  void* m[MT_MAX];
  void* v[MT_MAX];
  void* plow[MT_MAX];
  int64_t size[MT_MAX];
  int32_t chunk_start[MT_MAX + 1];  // prefix sum of chunks per tensor
  int32_t meta[MT_MAX];             // bits 0-7: scalar elements before the aligned body;
                                    // bit 8: vector accesses allowed
  int32_t n;
  int32_t chunk;                    // elements per workgroup (a multiple of 8)
};

__device__ __forceinline__ int head_of(const MtTable& t, int i) { return t.meta[i] & 0xff; }
__device__ __forceinline__ bool vec_ok_of(const MtTable& t, int i) { return (t.meta[i] & 0x100) != 0; }

__device__ __forceinline__ int find_tensor(const MtTable& t, int block) {
  int lo = 0, hi = t.n;  // chunk_start[lo] <= block < chunk_start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.chunk_start[mid] <= block) lo = mid; else hi = mid;
  }
  return lo;
}

template <int DT> struct Lowp;
template <> struct Lowp<AXN_BF16> {
  typedef uint16_t raw;
  __device__ static float to_float(raw x) { return __uint_as_float((uint32_t)x << 16); }
  __device__ static raw from_float(float f) {
    return __builtin_bit_cast(uint16_t, (__bf16)f);
  }
  __device__ static bool nonfinite(raw x) { return (x & 0x7F80u) == 0x7F80u; }
};
template <> struct Lowp<AXN_F16> {
  typedef uint16_t raw;
  __device__ static float to_float(raw x) { return (float)__builtin_bit_cast(_Float16, x); }
  __device__ static raw from_float(float f) {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
  __device__ static bool nonfinite(raw x) { return (x & 0x7C00u) == 0x7C00u; }
};
template <> struct Lowp<AXN_F32> {
  typedef uint32_t raw;
  __device__ static float to_float(raw x) { return __uint_as_float(x); }
  __device__ static raw from_float(float f) { return __float_as_uint(f); }
  __device__ static bool nonfinite(raw x) { return (x & 0x7F800000u) == 0x7F800000u; }
};

// Element range [begin, end) of tensor `t` owned by chunk `c`.  Chunk 0 also
// owns the scalar head [0, head).
struct Range {
  int64_t begin, end;
};
__device__ __forceinline__ Range chunk_range(const MtTable& tab, int t, int c) {
  const int64_t head = head_of(tab, t);
  Range r;
  r.begin = head + (int64_t)c * tab.chunk;
  r.end = r.begin + tab.chunk;
  if (r.end > tab.size[t]) r.end = tab.size[t];
  if (r.begin > r.end) r.begin = r.end;
  return r;
}

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

// One tensor's row of the table, in scalar registers.
struct TensorRow {
  const void* g;
  float* p;
  float* m;
  float* v;
  void* plow;
  int64_t size;
  int first_chunk;
  int meta;
};

// The row of the tensor that owns chunk `block`, through the scalar cache only: three
// pivots pick a quarter of the table, fifteen scalar compares on that quarter's starts pick
// the tensor, its row follows - three rounds of scalar loads from the argument block,
// which every wave of the launch repeats and the scalar cache holds.  Rows past the last
// tensor start at 2^31 - 1, which no chunk index reaches.  (Fetching row i in lane i with
// vector loads and voting is one round only, but those loads queue behind the streaming
// loads of the CU's other waves: 5.9 against 6.3 TB/s for the update.)
__device__ __forceinline__ TensorRow row_by_scalar_search(const MtTable& tab, int block) {
  static_assert(MT_MAX == 64, "four quarters of sixteen rows");
  // start <= block as the sign bit of start - block - 1 (both in [0, 2^31)): scalar adds only
  auto at_or_before = [block](int start) -> int { return (int)((uint32_t)(start - block - 1) >> 31); };
  const int q = at_or_before(tab.chunk_start[16]) + at_or_before(tab.chunk_start[32]) +
                at_or_before(tab.chunk_start[48]);
  const int base = q * 16;
  int t = base;
#pragma unroll
  for (int j = 1; j < 16; ++j) t += at_or_before(tab.chunk_start[base + j]);
  TensorRow r;
  r.g = tab.g[t];
  r.p = (float*)tab.p[t];
  r.m = (float*)tab.m[t];
  r.v = (float*)tab.v[t];
  r.plow = tab.plow[t];
  r.size = tab.size[t];
  r.first_chunk = tab.chunk_start[t];
  r.meta = tab.meta[t];
  return r;
}

// What the update's rate hangs on, measured on MI355X (1.3e9 elements, 64 tensors, 28 bytes
// per element; 6.5 to 6.6 TB/s as it stands):
//  - every access a wave makes covers consecutive bytes (one 4-element vector per lane:
//    16 bytes of each fp32 stream, 8 of each 16-bit one); loads non-temporal, stores
//    non-temporal and written through (nt + sc1: 1 to 2 % over nt alone, 10 % over plain
//    stores); 8 elements per lane in one access lose 6 %, cached loads of the state 13 %;
//  - all loads of a wave in front of its first store, and a wave that ends after its
//    stores: a wave that loops waits for its own stores before its next loads return
//    (the memory counter is in order; 16 trips per wave lose 6 %);
//  - one chunk per workgroup, handed out by the dispatcher in order, so that the chip
//    works on one compact window of every stream; resident workgroups that stride over
//    the chunks lose 8 to 12 %;
//  - FEWER waves in flight than the registers allow: with all 32 one-wave workgroups of a
//    CU resident the five streams thrash one another in the memory system (5.7 TB/s);
//    ten or eleven waves of one vector per lane are the best found (14 to 16 KB reserved
//    per workgroup: within 0.5 %; 12 KB: -2 %, 18 KB: -2.5 %).  The launch reserves ADAM_LDS
//    bytes of LDS per workgroup, which the kernel never touches, to hold the count there.
//    Several vectors per lane (ADAM_VECS) need fewer waves and make a skipped step cheaper
//    (1.27 M instead of 5.1 M workgroups that leave at once), but move 6 % less;
//  - a short way from the wave's start to its loads, because with few waves nothing hides
//    it: the table lookup stays on the scalar path, the scan result is loaded beside it,
//    not in front of it, and the accesses are buffer accesses (one descriptor per stream
//    in scalar registers, one 32-bit offset per lane: +3 to 4 % over 64-bit addresses
//    computed per lane).
template <int GDT, int PDT, bool HAS_PLOW, class Math>
__device__ __forceinline__ void update_chunk(const TensorRow& row, int b, int found_inf, float gmul, Math math) {
  typedef typename Lowp<GDT>::raw graw;
  typedef typename Lowp<PDT>::raw praw;
  const int tid = threadIdx.x;
  const int c = b - row.first_chunk;
  // Overflow: the whole step is skipped.  As an empty range rather than an early return,
  // so that the scan result's load runs beside the table's and not in front of it.
  const int head = found_inf != 0 ? 0 : row.meta & 0xff;
  const int64_t size = found_inf != 0 ? 0 : row.size;
  Range rg;
  rg.begin = head + (int64_t)c * ADAM_CHUNK;
  rg.end = rg.begin + ADAM_CHUNK;
  if (rg.end > size) rg.end = size;
  if (rg.begin > rg.end) rg.begin = rg.end;
  const void* g = row.g;
  float* p = row.p;
  float* m = row.m;
  float* v = row.v;
  void* plow = row.plow;

  auto one = [&](int64_t i) {
    float pp = p[i], mm = m[i], vv = v[i];
    math(Lowp<GDT>::to_float(((const graw*)g)[i]), pp, mm, vv, gmul);
    p[i] = pp;
    m[i] = mm;
    v[i] = vv;
    if (HAS_PLOW) ((praw*)plow)[i] = Lowp<PDT>::from_float(pp);
  };

  if (row.meta & 0x100) {
    if (c == 0 && tid < head) one(tid);
    const int nvec = (int)((rg.end - rg.begin) / ADAM_VEC);
    // ADAM_VECS vectors per lane, ADAM_THREADS vectors apart (every access of the wave
    // covers consecutive bytes), all loads in front of the first store.  Vector by vector
    // (g p m v, g p m v, ...); stream by stream (p p p p, m m m m, ...) measured the same on
    // constant data and 2 % slower on random data.
    // Each stream of the chunk is a buffer of exactly the bytes of its nvec vectors: the
    // hardware drops the accesses of the lanes behind the end (loads return zero, stores
    // do nothing), so a ragged last chunk runs the same code, and a lane needs one 32-bit
    // offset per access instead of a 64-bit address.
    constexpr int GSZ = (int)sizeof(graw), PSZ = (int)sizeof(praw);
    auto stream = [&](const void* base, int elem) {
      return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + rg.begin * elem), 0,
                                               nvec * ADAM_VEC * elem, 0x00020000);
    };
    if (nvec > 0) {   // (a skipped step's waves leave here)
    const __amdgpu_buffer_rsrc_t bg = stream(g, GSZ), bp = stream(p, 4), bm = stream(m, 4),
                                 bv = stream(v, 4), bl = stream(HAS_PLOW ? plow : p, PSZ);
    graw gr[ADAM_VECS][4];
    f32x4 pp[ADAM_VECS], mm[ADAM_VECS], vv[ADAM_VECS];
#pragma unroll
    for (int k = 0; k < ADAM_VECS; ++k) {
      const int e0 = (tid + k * ADAM_THREADS) * ADAM_VEC;
      if (GSZ == 2) {
        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(bg, e0 * 2, 0, ADAM_LOAD_POLICY));
        gr[k][0] = (graw)(w[0] & 0xFFFFu);
        gr[k][1] = (graw)(w[0] >> 16);
        gr[k][2] = (graw)(w[1] & 0xFFFFu);
        gr[k][3] = (graw)(w[1] >> 16);
      } else {
        const u32x4 w = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(bg, e0 * 4, 0, ADAM_LOAD_POLICY));
#pragma unroll
        for (int e = 0; e < 4; ++e) gr[k][e] = (graw)w[e];
      }
      pp[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bp, e0 * 4, 0, ADAM_LOAD_POLICY));
      mm[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bm, e0 * 4, 0, ADAM_LOAD_POLICY));
      vv[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(bv, e0 * 4, 0, ADAM_LOAD_POLICY));
    }
    __builtin_amdgcn_sched_barrier(0);   // every load is issued before the arithmetic of the first vector
#pragma unroll
    for (int k = 0; k < ADAM_VECS; ++k) {
      const int e0 = (tid + k * ADAM_THREADS) * ADAM_VEC;
      praw pl[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float pe = pp[k][e], me = mm[k][e], ve = vv[k][e];
        math(Lowp<GDT>::to_float(gr[k][e]), pe, me, ve, gmul);
        pp[k][e] = pe;
        mm[k][e] = me;
        vv[k][e] = ve;
        if (HAS_PLOW) pl[e] = Lowp<PDT>::from_float(pe);
      }
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, pp[k]), bp, e0 * 4, 0, ADAM_STORE_POLICY);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, mm[k]), bm, e0 * 4, 0, ADAM_STORE_POLICY);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, vv[k]), bv, e0 * 4, 0, ADAM_STORE_POLICY);
      if (HAS_PLOW) {
        if (PSZ == 2) {
          u32x2 w;
          w[0] = (uint32_t)pl[0] | ((uint32_t)pl[1] << 16);
          w[1] = (uint32_t)pl[2] | ((uint32_t)pl[3] << 16);
          __builtin_amdgcn_raw_buffer_store_b64(w, bl, e0 * 2, 0, ADAM_STORE_POLICY);
        } else {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = (uint32_t)pl[e];
          __builtin_amdgcn_raw_buffer_store_b128(w, bl, e0 * 4, 0, ADAM_STORE_POLICY);
        }
      }
    }
    }
    const int64_t tail = rg.begin + (int64_t)nvec * ADAM_VEC;
    if (tail + tid < rg.end) one(tail + tid);
  } else {
    const int64_t b0 = (c == 0) ? 0 : rg.begin;
    for (int64_t i = b0 + tid; i < rg.end; i += ADAM_THREADS) one(i);
  }
}

// ------------------------------------------------------------- host side ----
int dtype_size(int dt) { return dt == AXN_F32 ? 4 : 2; }

// Number of leading scalar elements after which every given pointer of a
// tensor is 16-byte aligned, or -1 when no common count exists.  The pointer
// with the narrowest element decides the count; the others must agree.
int common_head(const void* const* ptrs, const int* elem_sizes, int count) {
  int best = 0;
  for (int i = 0; i < count; ++i) {
    if (ptrs[i] == nullptr) continue;
    const uintptr_t a = (uintptr_t)ptrs[i];
    const int es = elem_sizes[i];
    if (a % es != 0) return -1;
    const int h = (int)(((16 - a % 16) % 16) / es);
    if (h > best) best = h;
  }
  for (int i = 0; i < count; ++i) {
    if (ptrs[i] == nullptr) continue;
    const uintptr_t a = (uintptr_t)ptrs[i] + (uintptr_t)best * elem_sizes[i];
    if (a % 16 != 0) return -1;
  }
  // Prefer a head after which every pointer sits on a 128-byte cache line, so that
  // the chunks of different workgroups do not share lines (views at one common
  // element offset into line-aligned flat buffers always have one, of at most 63
  // elements).  Steps of 8 elements keep the 16-byte alignment found above.
  for (int h = best; h < 64; h += 8) {
    bool all = true;
    for (int i = 0; i < count && all; ++i)
      if (ptrs[i] != nullptr)
        all = ((uintptr_t)ptrs[i] + (uintptr_t)h * elem_sizes[i]) % 128 == 0;
    if (all) return h;
  }
  return best;
}

struct Group {
  MtTable tab;
  int blocks;
};

// Walks the tensor list in launch groups and hands each filled argument table to `emit`, which
// returns a status; the first non-zero status ends the walk.  A group has at most MT_MAX tensors
// and below 2^32 threads, `threads` to a chunk: a launch of more wraps without an error.
// `ptr_sets[k][i]` is pointer k of tensor i (k = 0 is always the gradient).  Nothing is
// allocated: the one table lives on the stack.
template <class Emit>
int for_each_group(const void* const* const* ptr_sets, const int* elem_sizes, int nsets,
                   const int64_t* h_sizes, int64_t n, int chunk, int threads, Emit&& emit) {
  const int64_t most = 0xffffffffLL / threads;
  Group cur;
  cur.tab = MtTable();
  cur.blocks = 0;
  int k = 0;
  auto flush = [&]() -> int {
    if (k == 0) return AXN_OK;
    cur.tab.n = k;
    cur.tab.chunk = chunk;
    // past the last tensor: a start no workgroup index reaches, so that a lookup need
    // not know the count
    for (int j = k; j <= MT_MAX; ++j) cur.tab.chunk_start[j] = j == k ? cur.blocks : 0x7fffffff;
    const int rc = emit(cur);
    cur.tab = MtTable();
    cur.blocks = 0;
    k = 0;
    return rc;
  };
  for (int64_t i = 0; i < n; ++i) {
    const int64_t sz = h_sizes[i];
    if (sz == 0) continue;
    const void* ptrs[5] = {nullptr, nullptr, nullptr, nullptr, nullptr};
    for (int s = 0; s < nsets; ++s) ptrs[s] = ptr_sets[s] ? ptr_sets[s][i] : nullptr;
    int head = common_head(ptrs, elem_sizes, nsets);
    const bool vec_ok = head >= 0;
    if (!vec_ok) head = 0;
    if (head > sz) head = (int)sz;
    const int64_t body = sz - head;
    int64_t chunks = (body + chunk - 1) / chunk;
    if (chunks == 0) chunks = 1;  // the head still needs a workgroup
    if (chunks > most) {
      set_error("multi-tensor: tensor %lld has too many elements (%lld)",
                (long long)i, (long long)sz);
      return AXN_ELIMIT;
    }
    if (k == MT_MAX || cur.blocks + chunks > most) {
      const int rc = flush();
      if (rc != AXN_OK) return rc;
    }
    cur.tab.g[k] = ptrs[0];
    cur.tab.p[k] = const_cast<void*>(ptrs[1]);
    cur.tab.m[k] = const_cast<void*>(ptrs[2]);
    cur.tab.v[k] = const_cast<void*>(ptrs[3]);
    cur.tab.plow[k] = const_cast<void*>(ptrs[4]);
    cur.tab.size[k] = sz;
    cur.tab.chunk_start[k] = cur.blocks;
    cur.tab.meta[k] = head | (vec_ok ? 0x100 : 0);
    cur.blocks += (int)chunks;
    ++k;
  }
  return flush();
}

}  // namespace
}  // namespace axn
