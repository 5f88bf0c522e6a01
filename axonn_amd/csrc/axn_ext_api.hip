// The C ABI of axn_ext.h: argument checks and dispatch only.
#include <algorithm>
#include <new>

#include "axn_checks.h"
#include "axn_internal.h"

using namespace axn;

namespace {

bool aligned_to(const void* p, size_t bytes) { return (uintptr_t)p % bytes == 0; }
int elem_bytes(int dtype) { return dtype == AXN_F32 ? 4 : 2; }

int check_norm(const char* name, int dtype, int param_dtype, int64_t M, int64_t N) {
  REQUIRE(known_dtype(dtype), AXN_EINVAL, "%s: unknown dtype %d", name, dtype);
  REQUIRE(param_dtype == dtype || param_dtype == AXN_F32, AXN_EINVAL, "%s: parameters must have the rows' type or fp32",
          name);
  REQUIRE(M >= 0 && N >= 1, AXN_EINVAL, "%s: M must be >= 0 and N >= 1 (got %lld, %lld)", name, (long long)M, (long long)N);
  REQUIRE(M <= 0x7fffffff && N <= 0x7fffffff, AXN_ELIMIT, "%s: M and N must be below 2^31", name);
  return AXN_OK;
}

int check_rows(const char* name, const char* what, const void* p, int bytes, int64_t M, int64_t N, int64_t ld) {
  REQUIRE(p != nullptr, AXN_EINVAL, "%s: %s is null", name, what);
  REQUIRE(aligned_to(p, bytes), AXN_EALIGN, "%s: %s is not aligned to its element size", name, what);
  REQUIRE(ld >= N || M == 1, AXN_EINVAL, "%s: row stride of %s is smaller than the row", name, what);
  return AXN_OK;
}

int check_param(const char* name, const char* what, const void* p, int bytes) {
  REQUIRE(aligned_to(p, bytes), AXN_EALIGN, "%s: %s is not aligned to its element size", name, what);
  return AXN_OK;
}

#define CHECK(call)          \
  do {                       \
    const int rc__ = (call); \
    if (rc__) return rc__;   \
  } while (0)

// One list of a step's tensors: `bytes` for an element, or for every block of them begun.
struct List {
  const char* what;
  const void* const* at;
  int64_t bytes;
  bool blocks;
  uintptr_t begin, end;   // all of the list lies in between
  uintptr_t from(int64_t i) const { return (uintptr_t)at[i]; }
  uintptr_t to(int64_t i, const int64_t* h_sizes) const {
    return from(i) + (uintptr_t)((blocks ? ceil_div(h_sizes[i], AXN_ADAMW8_BLOCK) : h_sizes[i]) * bytes);
  }
};
struct Span {
  uintptr_t begin, end;
  int list;
  int64_t tensor;
};

// Two written tensors that share bytes would be written by two workgroups at once, a gradient that shares
// some with them would be read by one after another has written it.  A gradient may lie where its own weight
// or copy does, element for element: a lane reads it before it writes there.
// Lists in ascending order that lie apart as a whole, as the views of flat buffers do, are done in one walk
// each.  Lists: gradients, weights, two of the moments, copies.  Two tensors of one list are named first.
int check_apart(const char* name, List* lists, int count, const int64_t* h_sizes, int64_t n) {
  bool ascending = true, apart = true;
  for (int l = 0; l < count; ++l) {
    List& a = lists[l];
    uintptr_t last = 0;
    a.begin = ~(uintptr_t)0, a.end = 0;
    for (int64_t i = 0; i < n; ++i) {
      if (h_sizes[i] == 0) continue;
      const uintptr_t begin = a.from(i), end = a.to(i, h_sizes);
      ascending = ascending && (l == 0 || begin >= last);   // (gradients are read: two may be the same)
      last = end;
      a.begin = std::min(a.begin, begin), a.end = std::max(a.end, end);
    }
    for (int k = 0; k < l; ++k) apart = apart && (a.end <= lists[k].begin || lists[k].end <= a.begin);
  }
  if (ascending && apart) return AXN_OK;
  Span* spans = new (std::nothrow) Span[(size_t)n * (count - 1)];
  REQUIRE(spans != nullptr, AXN_ELIMIT, "%s: no host memory to order %lld tensors", name, (long long)n);
  int64_t used = 0;
  for (int l = 1; l < count; ++l)
    for (int64_t i = 0; i < n; ++i)
      if (h_sizes[i] != 0) spans[used++] = {lists[l].from(i), lists[l].to(i, h_sizes), l, i};
  std::sort(spans, spans + used, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  // a pair that overlaps: of the written ones two that follow one another (of one list, if there are such)
  int one = 0, other = 0;
  for (int64_t i = 1; i < used; ++i)
    if (spans[i - 1].end > spans[i].begin && (one == 0 || spans[i - 1].list == spans[i].list)) {
      one = spans[i - 1].list, other = spans[i].list;
      if (one == other) break;
    }
  bool gradient = false;
  for (int64_t i = 0; i < n && one == 0; ++i) {
    if (h_sizes[i] == 0) continue;
    const uintptr_t begin = lists[0].from(i), end = lists[0].to(i, h_sizes);
    // (written ones are apart by now, so that their ends ascend too)
    const Span* s = std::upper_bound(spans, spans + used, begin, [](uintptr_t at, const Span& a) { return at < a.end; });
    if (s == spans + used || s->begin >= end) continue;
    const bool own = (s->list == 1 || s->list == 4) && s->begin == begin && s->end == end && s->tensor == i;
    if (!own) one = s->list, gradient = true;
  }
  delete[] spans;
  REQUIRE(!gradient, AXN_EINVAL, "%s: a tensor of g and one of %s overlap", name, lists[one].what);
  REQUIRE(one == 0 || one != other, AXN_EINVAL, "%s: two tensors of %s overlap", name, lists[one].what);
  REQUIRE(one == 0, AXN_EINVAL, "%s: a tensor of %s and one of %s overlap", name, lists[one].what, lists[other].what);
  return AXN_OK;
}

}  // namespace

extern "C" {

int axn_ext_abi_version(void) { return AXN_EXT_ABI_VERSION; }

int axn_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* sum,
                       float* mean, float* rstd, int dtype, int param_dtype, int64_t M, int64_t N, int64_t ldx,
                       int64_t ldr, float eps, void* stream) {
  const char* name = "axn_layer_norm_fwd";
  CHECK(check_norm(name, dtype, param_dtype, M, N));
  REQUIRE(eps >= 0.0f, AXN_EINVAL, "%s: eps must be >= 0", name);
  REQUIRE((mean == nullptr) == (rstd == nullptr), AXN_EINVAL, "%s: mean and rstd come together", name);
  REQUIRE((residual == nullptr) == (sum == nullptr), AXN_EINVAL, "%s: residual and sum come together", name);
  if (M == 0) return AXN_OK;
  const int es = elem_bytes(dtype), ps = elem_bytes(param_dtype);
  CHECK(check_rows(name, "x", x, es, M, N, ldx));
  if (residual) CHECK(check_rows(name, "residual", residual, es, M, N, ldr));
  CHECK(check_rows(name, "y", y, es, M, N, N));
  CHECK(check_param(name, "sum", sum, es));
  CHECK(check_param(name, "weight", weight, ps));
  CHECK(check_param(name, "bias", bias, ps));
  CHECK(check_param(name, "mean", mean, 4));
  CHECK(check_param(name, "rstd", rstd, 4));
  return launch_layer_norm_fwd(x, residual, weight, bias, y, sum, mean, rstd, dtype, param_dtype != dtype, M, N, ldx, ldr,
                               eps, (hipStream_t)stream);
}

size_t axn_layer_norm_bwd_workspace_bytes(int64_t M, int64_t N) {
  if (M > 0x7fffffff || N > 0x7fffffff) return 0;
  return layer_norm_bwd_workspace_bytes(M, N);
}

int axn_layer_norm_bwd(const void* dy, const void* h, const void* weight, const float* mean, const float* rstd,
                       const void* dsum, void* dx, void* dweight, void* dbias, int dtype, int param_dtype, int64_t M,
                       int64_t N, int64_t lddy, int64_t ldh, int64_t lddsum, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const char* name = "axn_layer_norm_bwd";
  CHECK(check_norm(name, dtype, param_dtype, M, N));
  REQUIRE(dx || dweight || dbias, AXN_EINVAL, "%s: nothing to compute", name);
  const int es = elem_bytes(dtype), ps = elem_bytes(param_dtype);
  CHECK(check_param(name, "dweight", dweight, ps));
  CHECK(check_param(name, "dbias", dbias, ps));
  if (M > 0) {
    CHECK(check_rows(name, "dy", dy, es, M, N, lddy));
    CHECK(check_rows(name, "h", h, es, M, N, ldh));
    if (dsum) CHECK(check_rows(name, "dsum", dsum, es, M, N, lddsum));
    CHECK(check_param(name, "weight", weight, ps));
    REQUIRE(mean && rstd, AXN_EINVAL, "%s: mean or rstd is null", name);
    CHECK(check_param(name, "mean", mean, 4));
    CHECK(check_param(name, "rstd", rstd, 4));
    CHECK(check_param(name, "dx", dx, es));
    if ((dweight || dbias) && layer_norm_bwd_workspace_bytes(M, N) > 0) {
      REQUIRE(workspace != nullptr && workspace_bytes >= layer_norm_bwd_workspace_bytes(M, N), AXN_EINVAL,
              "%s: workspace too small (%zu bytes given, %zu needed)", name, workspace_bytes,
              layer_norm_bwd_workspace_bytes(M, N));
      REQUIRE(aligned16(workspace), AXN_EALIGN, "%s: workspace must be 16-byte aligned", name);
    }
  }
  if (M == 0 && !dweight && !dbias) return AXN_OK;
  return launch_layer_norm_bwd(dy, h, weight, mean, rstd, dsum, M == 0 ? nullptr : dx, dweight, dbias, dtype,
                               param_dtype != dtype, M, N, lddy, ldh, lddsum, workspace, (hipStream_t)stream);
}

static int check_adamw(const char* name, const void* const* h_g, void* const* h_p, void* const* h_m, void* const* h_v,
                       void* const* h_plow, const int64_t* h_sizes, int64_t n, int g_dtype, int plow_dtype,
                       const axn_adamw_hparams* hp) {
  CHECK(check_sizes(name, h_sizes, n));
  REQUIRE(known_dtype(g_dtype), AXN_EINVAL, "%s: unknown gradient dtype %d", name, g_dtype);
  REQUIRE(h_plow == nullptr || plow_dtype == AXN_BF16 || plow_dtype == AXN_F16, AXN_EINVAL,
          "%s: low-precision copy must be bf16 or fp16", name);
  REQUIRE(hp != nullptr, AXN_EINVAL, "%s: hyper-parameters are null", name);
  REQUIRE(n == 0 || (h_g && h_p && h_m && h_v), AXN_EINVAL, "%s: null pointer array", name);
  CHECK(check_list(name, h_g, "g", h_sizes, n, elem_bytes(g_dtype)));
  CHECK(check_list(name, (const void* const*)h_p, "p", h_sizes, n, 4));
  if (h_plow != nullptr) CHECK(check_list(name, (const void* const*)h_plow, "p_lowp", h_sizes, n, 2));
  return AXN_OK;
}

int axn_mt_adamw(const void* const* h_g, void* const* h_p, void* const* h_m, void* const* h_v, void* const* h_plow,
                 const int64_t* h_sizes, int64_t n, int g_dtype, int plow_dtype, float inv_scale,
                 const axn_scan_result* scan, const axn_adamw_hparams* hp, void* stream) {
  const char* name = "axn_mt_adamw";
  CHECK(check_adamw(name, h_g, h_p, h_m, h_v, h_plow, h_sizes, n, g_dtype, plow_dtype, hp));
  CHECK(check_list(name, (const void* const*)h_m, "m", h_sizes, n, 4));
  CHECK(check_list(name, (const void* const*)h_v, "v", h_sizes, n, 4));
  List lists[] = {{"g", h_g, elem_bytes(g_dtype), false},
                  {"p", (const void* const*)h_p, 4, false},
                  {"m", (const void* const*)h_m, 4, false},
                  {"v", (const void* const*)h_v, 4, false},
                  {"p_lowp", (const void* const*)h_plow, 2, false}};
  CHECK(check_apart(name, lists, h_plow ? 5 : 4, h_sizes, n));
  return launch_mt_adamw(h_g, h_p, h_m, h_v, h_plow, h_sizes, n, g_dtype, h_plow ? plow_dtype : AXN_BF16, inv_scale, scan,
                         *hp, (hipStream_t)stream);
}

int axn_mt_adamw8(const void* const* h_g, void* const* h_p, void* const* h_codes, void* const* h_exponents,
                  void* const* h_plow, const int64_t* h_sizes, int64_t n, int g_dtype, int plow_dtype, float inv_scale,
                  uint64_t seed, const axn_scan_result* scan, const axn_adamw_hparams* hp, void* stream) {
  const char* name = "axn_mt_adamw8";
  CHECK(check_adamw(name, h_g, h_p, h_codes, h_exponents, h_plow, h_sizes, n, g_dtype, plow_dtype, hp));
  CHECK(check_list(name, (const void* const*)h_codes, "codes", h_sizes, n, 8));
  CHECK(check_list(name, (const void* const*)h_exponents, "exponents", h_sizes, n, 2));
  for (int64_t i = 0; i < n; ++i)
    REQUIRE(ceil_div(h_sizes[i], AXN_ADAMW8_BLOCK) < (1 << 26), AXN_ELIMIT, "%s: tensor %lld has too many elements (%lld)",
            name, (long long)i, (long long)h_sizes[i]);
  List lists[] = {{"g", h_g, elem_bytes(g_dtype), false},
                  {"p", (const void* const*)h_p, 4, false},
                  {"codes", (const void* const*)h_codes, 2 * AXN_ADAMW8_BLOCK, true},
                  {"exponents", (const void* const*)h_exponents, 2, true},
                  {"p_lowp", (const void* const*)h_plow, 2, false}};
  CHECK(check_apart(name, lists, h_plow ? 5 : 4, h_sizes, n));
  return launch_mt_adamw8(h_g, h_p, h_codes, h_exponents, h_plow, h_sizes, n, g_dtype, h_plow ? plow_dtype : AXN_BF16,
                          inv_scale, seed, scan, *hp, (hipStream_t)stream);
}

int axn_adamw8_moments(const void* codes, const void* exponents, void* m, void* v, int dtype, int64_t n, void* stream) {
  const char* name = "axn_adamw8_moments";
  REQUIRE(dtype == AXN_F32 || dtype == AXN_BF16, AXN_EINVAL, "%s: moments come as fp32 or bf16", name);
  REQUIRE(n >= 0, AXN_EINVAL, "%s: negative element count", name);
  if (n == 0) return AXN_OK;
  REQUIRE(m || v, AXN_EINVAL, "%s: nothing to compute", name);
  REQUIRE(codes && exponents, AXN_EINVAL, "%s: null pointer", name);
  REQUIRE(aligned_to(codes, 8) && aligned_to(exponents, 2) && aligned_to(m, elem_bytes(dtype)) &&
              aligned_to(v, elem_bytes(dtype)),
          AXN_EALIGN, "%s: pointers must be aligned to 8 bytes (codes), 2 (exponents) and their elements", name);
  REQUIRE(n < (1LL << 40), AXN_ELIMIT, "%s: too many elements", name);
  return launch_adamw8_moments(codes, exponents, m, v, dtype, n, (hipStream_t)stream);
}

}  // extern "C"
