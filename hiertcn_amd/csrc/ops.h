// Shared by the sequence operators (glr.hip, seq_loss.hip, adamw.hip): errors, typed vector access, views.  Unlike the model kernels these take
// fp32, bfloat16 and IEEE half side by side in both library builds, so nothing here depends on HIERTCN_F16.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hiertcn_ops.h"

int ops_fail(int code, const char* fmt, ...);   // sets this thread's message, returns code
#define OPS_TRY(expr)                                                                                                                        \
  do {                                                                                                                                       \
    hipError_t e_ = (expr);                                                                                                                  \
    if (e_ != hipSuccess) return ops_fail(HIERTCN_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__);       \
  } while (0)

// workgroups of a launch, at most: HIP counts its threads in 32 bits
constexpr int64_t ops_most_groups(int threads) { return 0xffffffffll / threads; }

static inline int ops_size(int dtype) { return dtype == HIERTCN_FP32 ? 4 : 2; }
static inline bool ops_dtype_ok(int dtype) { return dtype >= HIERTCN_FP32 && dtype <= HIERTCN_FP16; }

// A [nb][nt][nd] view with element strides (nd contiguous).  Host side, for the overlap checks.
struct OpsView {
  const char* p; int64_t nb, nt, nd, sb, st; int es;
  int64_t extent() const { return nb && nt && nd ? ((nb - 1) * sb + (nt - 1) * st + nd) * es : 0; }
};
static inline OpsView ops_flat(const void* p, int64_t n, int es) { return {static_cast<const char*>(p), 1, 1, n, 0, 0, es}; }
// rows of the view do not overlap one another (an output may not hold one place twice)
static inline bool ops_rows_apart(const OpsView& v) {
  if (v.nb <= 1 && v.nt <= 1) return true;
  if (v.nb <= 1) return v.st >= v.nd;
  if (v.nt <= 1) return v.sb >= v.nd;
  return (v.st >= v.nd && v.sb >= (v.nt - 1) * v.st + v.nd) || (v.sb >= v.nd && v.st >= (v.nb - 1) * v.sb + v.nd);
}
// true if the two views may share a place.  Rows of one buffer side by side (the halves of a [B][T][2 D] projection) are told apart.
static inline bool ops_overlap(const OpsView& a, const OpsView& b) {
  if (!a.p || !b.p || !a.extent() || !b.extent()) return false;
  if (a.p + a.extent() <= b.p || b.p + b.extent() <= a.p) return false;
  const OpsView& lo = a.p <= b.p ? a : b;
  const OpsView& hi = a.p <= b.p ? b : a;
  if (a.es != b.es || a.nb != b.nb || a.nt != b.nt || a.nd != b.nd || a.sb != b.sb || a.st != b.st || !ops_rows_apart(a)) return true;
  // both strides are multiples of the smaller one: two rows are d + k * small apart, nearest for the d % small at hand
  const int64_t small = (a.nb <= 1 ? a.st : a.nt <= 1 ? a.sb : a.sb < a.st ? a.sb : a.st) * a.es, row = a.nd * a.es;
  if (small <= 0 || (a.nb > 1 && a.sb * a.es % small) || (a.nt > 1 && a.st * a.es % small)) return true;
  const int64_t r = (hi.p - lo.p) % small;
  return !(r >= row && small - r >= row);
}

// ---- device side ----------------------------------------------------------------------------------------------------------------------------
template <int VEC>
struct alignas(4 * VEC) OpsF { float v[VEC]; };
template <int VEC>
struct alignas(2 * VEC) OpsH { uint16_t v[VEC]; };

__device__ __forceinline__ float ops_h2f(uint16_t u, int dt) {
  return dt == HIERTCN_BF16 ? __builtin_bit_cast(float, (uint32_t)u << 16) : (float)__builtin_bit_cast(_Float16, u);
}
__device__ __forceinline__ uint16_t ops_f2h(float f, int dt) {   // round to nearest, ties to even
  if (dt == HIERTCN_BF16) { __bf16 b = (__bf16)f; return __builtin_bit_cast(uint16_t, b); }
  _Float16 h = (_Float16)f;
  return __builtin_bit_cast(uint16_t, h);
}
// VEC elements of type DT at element offset `off` <-> fp32 registers.  The address is a multiple of VEC elements.
template <int DT, int VEC>
__device__ __forceinline__ void ops_ld(const void* __restrict__ p, int64_t off, float (&o)[VEC]) {
  if constexpr (DT == HIERTCN_FP32) {
    const OpsF<VEC> x = *reinterpret_cast<const OpsF<VEC>*>(static_cast<const float*>(p) + off);
#pragma unroll
    for (int i = 0; i < VEC; i++) o[i] = x.v[i];
  } else {
    const OpsH<VEC> x = *reinterpret_cast<const OpsH<VEC>*>(static_cast<const uint16_t*>(p) + off);
#pragma unroll
    for (int i = 0; i < VEC; i++) o[i] = ops_h2f(x.v[i], DT);
  }
}
typedef float ops_f4 __attribute__((ext_vector_type(4)));
template <bool PAST, typename T>
__device__ __forceinline__ void ops_put(void* p, const T& x) {
  if constexpr (PAST && sizeof(T) == 16) __builtin_nontemporal_store(__builtin_bit_cast(ops_f4, x), static_cast<ops_f4*>(p));
  else *static_cast<T*>(p) = x;
}
// PAST: a store that leaves the caches to others, 16 bytes wide (and an ordinary one at any other width)
template <int DT, int VEC, bool PAST = false>
__device__ __forceinline__ void ops_st(void* __restrict__ p, int64_t off, const float (&o)[VEC]) {
  if constexpr (DT == HIERTCN_FP32) {
    OpsF<VEC> x;
#pragma unroll
    for (int i = 0; i < VEC; i++) x.v[i] = o[i];
    ops_put<PAST>(static_cast<float*>(p) + off, x);
  } else {
    OpsH<VEC> x;
#pragma unroll
    for (int i = 0; i < VEC; i++) x.v[i] = ops_f2h(o[i], DT);
    ops_put<PAST>(static_cast<uint16_t*>(p) + off, x);
  }
}
// the same in two steps, so that many loads can be in flight before the first is converted
template <int DT, int VEC>
struct OpsRaw { typedef OpsH<VEC> type; };
template <int VEC>
struct OpsRaw<HIERTCN_FP32, VEC> { typedef OpsF<VEC> type; };
template <int DT, int VEC>
__device__ __forceinline__ void ops_cvt(const typename OpsRaw<DT, VEC>::type& x, float (&o)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    if constexpr (DT == HIERTCN_FP32) o[i] = x.v[i];
    else o[i] = ops_h2f(x.v[i], DT);
  }
}
// ---- words between workgroups: 64 bits that are their own flag, all ones until written; one store or load that goes past the L2s --------------------
constexpr uint64_t OPS_NOTHING = ~0ull;
__device__ __forceinline__ uint64_t ops_word(float lo, float hi) {      // (a NaN in the low half is stored as the canonical one: no result looks like nothing)
  if (lo != lo) lo = __builtin_bit_cast(float, 0x7fc00000u);
  return (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo);
}
__device__ __forceinline__ float ops_low(uint64_t v) { return __builtin_bit_cast(float, (uint32_t)v); }
__device__ __forceinline__ float ops_high(uint64_t v) { return __builtin_bit_cast(float, (uint32_t)(v >> 32)); }
__device__ __forceinline__ void ops_publish(uint64_t* p, uint64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// Waits for a word.  A wait that cannot end gives up after `polls` looks, or soon after another has (*gave_up is set then): the word is a pair of NaNs.
constexpr unsigned OPS_POLLS = 1u << 22;      // some seconds; a word that is on its way takes microseconds
__device__ __forceinline__ uint64_t ops_await(const uint64_t* p, unsigned* gave_up, unsigned polls) {
  uint64_t v;
  unsigned n = 0;
  while ((v = __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == OPS_NOTHING) {
    if (++n > polls || (n % 64 == 0 && __hip_atomic_load(gave_up, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))) {
      __hip_atomic_store(gave_up, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return ops_word(__builtin_nanf(""), __builtin_nanf(""));
    }
    __builtin_amdgcn_s_sleep(1);
  }
  return v;
}
// The ticket of a workgroup: the order in which workgroups START, whatever order they are dispatched in.  `place`: LDS.  One barrier.
__device__ __forceinline__ unsigned ops_ticket(unsigned* counter, unsigned* place) {
  if (threadIdx.x == 0) *place = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return (unsigned)__builtin_amdgcn_readfirstlane((int)*place);
}
// e^x for x <= 0 through v_exp_f32 (one ulp).  The product x log2 e is rounded: |x| half steps of the result, too few to matter behind a 16-bit rounding.
__device__ __forceinline__ float ops_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
// The same to 3 half steps and |x| / 20: with t = x log2 e as rounded, e^x = 2^t e^(x - t ln 2), whose second factor is 1 + (x - t ln 2) to 2^-33.
__device__ __forceinline__ float ops_exp_fp32(float x) {
  const float t = x * 1.4426950408889634f, e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, __builtin_amdgcn_fmed3f(fmaf(t, -0.6931471805599453f, x), -1.f, 1.f), e);      // (t may be -inf, and the inner one infinite or NaN: e is 0 then)
}
// the one of the two that operands of type DT are worth
template <int DT>
__device__ __forceinline__ float ops_exp_of(float x) { return DT == HIERTCN_FP32 ? ops_exp_fp32(x) : ops_exp(x); }
