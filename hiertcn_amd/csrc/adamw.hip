// AdamW over many tensors at once, states in 32 or in 8 bits (include/hiertcn_ops.h).
//
// A wave owns 256 consecutive elements of a tensor, four to a lane: exactly a block of the 8-bit states, so a block's new scale is a maximum over a
// wave and its codes never leave the registers between decoding and encoding.  The tensors of a launch travel as kernel arguments (pointers and
// the first workgroup of each), so nothing is uploaded and nothing is kept between calls.
//
// 8-bit states.  m = sign (q / 127)^2 scale and sqrt(v) = (q / 255)^2 scale: relative steps of 2 / q near the top and a range of 1.6e4 (m) and 6.5e4
// (sqrt v).  A step of Adam changes v by about (1 - b2) = 1e-3 of itself where a code is 4 / q >= 1.6e-2 of v wide, so rounding to nearest would
// never move it; a code is rounded up with probability (x - a) / (b - a) between its neighbours' VALUES a <= x < b (of |m| and of v), which keeps the
// expectation.  The arithmetic up to the codes is single operations in fp32 without contraction, so that any other implementation of the formula
// that rounds every operation gets the same codes.
#include <math.h>

#include "ops.h"

namespace {

constexpr int NT = 256, BLOCK = 256;     // threads of a workgroup; elements of a block (one wave, four to a lane)
constexpr int PER_WG = NT / 64;          // blocks of a workgroup
constexpr int MAX_TENSORS = 40;          // of a launch: 40 descriptors fit the 4 KB of kernel arguments

struct Batch {
  hiertcn_adamw_tensor_t t[MAX_TENSORS];
  uint32_t first[MAX_TENSORS + 1];       // first workgroup of a tensor
  int n;
  float b1, c1, b2, c2, step, root, eps, gscale;      // c = 1 - b
  float decay[MAX_TENSORS];              // 1 - lr * weight_decay
  const float* gscale_dev;
  uint32_t key;                          // of the random bits, without the tensor's share
  uint64_t wide;                         // bit i: tensor i's addresses allow four elements at a time
};
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

__device__ __forceinline__ uint32_t mix(uint64_t e, uint32_t key) {
  uint32_t x = (uint32_t)e * 0x9E3779B1u + key + (uint32_t)(e >> 32) * 0x1F83D9ABu;
  x = (x ^ (x >> 16)) * 0x3C6EF373u;
  x = (x ^ (x >> 15)) * 0x510E527Fu;
  return x ^ (x >> 16);
}

// where a lane's four elements of a block lie: neighbours where the addresses allow it, else 64 apart
struct Lane {
  int64_t base;
  int step, n;                           // element i: base + i * step; the first n exist
};
__device__ __forceinline__ Lane lane_of(int64_t block, int64_t numel, bool wide) {
  const int lane = threadIdx.x & 63;
  Lane l;
  l.step = wide ? 1 : 64;
  l.base = block * BLOCK + (wide ? lane * 4 : lane);
  const int64_t left = numel - l.base;
  l.n = left <= 0 ? 0 : wide ? (left < 4 ? (int)left : 4) : (int)((left + 63) / 64 < 4 ? (left + 63) / 64 : 4);
  return l;
}
template <typename T>
struct alignas(4 * sizeof(T)) Four { T v[4]; };
template <typename T>
__device__ __forceinline__ void load4(const void* p, const Lane& l, T (&o)[4]) {
  const T* q = static_cast<const T*>(p) + l.base;
  if (l.step == 1 && l.n == 4) {
    const Four<T> x = *reinterpret_cast<const Four<T>*>(q);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = x.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = i < l.n ? q[i * l.step] : T(0);
  }
}
template <typename T>
__device__ __forceinline__ void store4(void* p, const Lane& l, const T (&o)[4]) {
  T* q = static_cast<T*>(p) + l.base;
  if (l.step == 1 && l.n == 4) {
    Four<T> x;
#pragma unroll
    for (int i = 0; i < 4; i++) x.v[i] = o[i];
    *reinterpret_cast<Four<T>*>(q) = x;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < l.n) q[i * l.step] = o[i];
  }
}
__device__ __forceinline__ void load_grad(const hiertcn_adamw_tensor_t& t, const Lane& l, float (&g)[4]) {
  if (t.grad_dtype == HIERTCN_FP32) {
    load4<float>(t.grad, l, g);
  } else {
    uint16_t h[4];
    load4<uint16_t>(t.grad, l, h);
#pragma unroll
    for (int i = 0; i < 4; i++) g[i] = t.grad_dtype == HIERTCN_BF16 ? ops_h2f(h[i], HIERTCN_BF16) : ops_h2f(h[i], HIERTCN_FP16);
  }
}
__device__ __forceinline__ float wave_max(float x) {      // NaN wins
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float y = __shfl_xor(x, d);
    x = y > x || y != y ? y : x;
  }
  return x;
}
__device__ __forceinline__ float decode_m(int q, float scale) {
#pragma clang fp contract(off)
  const float f = (float)q * (1.f / 127.f);
  return f * fabsf(f) * scale;
}
__device__ __forceinline__ float decode_v(uint32_t q, float scale) {
#pragma clang fp contract(off)
  const float f = (float)q * (1.f / 255.f);
  const float x = f * f * scale;
  return x * x;
}
// code of a magnitude: the largest a with a <= r, or the next one up with the probability that keeps the expectation
template <bool SQUARED>
__device__ __forceinline__ int encode(float mag, float inv, uint32_t bits) {
#pragma clang fp contract(off)
  constexpr float TOP = SQUARED ? 255.f : 127.f;
  float r = mag * inv;
  const float q = fminf(floorf(sqrtf(r) * TOP), TOP - 1.f);
  float a = q * (1.f / TOP), b = (q + 1.f) * (1.f / TOP);
  a = a * a;
  b = b * b;
  if (SQUARED) {
    a = a * a;
    b = b * b;
    r = r * r;
  }
  const float u = (float)bits * 1.52587890625e-5f;
  const int code = (int)fmaxf(q, 0.f) + (r - a > u * (b - a) ? 1 : 0);
  return SQUARED && mag > 0.f && inv > 0.f && code < 1 ? 1 : code;
}
__device__ __forceinline__ float scale_of(float largest) { return largest < 7.888609052210118e-31f ? 0.f : largest; }      // 2^-100
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.f ? 1.f / scale : 0.f; }

__device__ __forceinline__ int tensor_of(const Batch& b, uint32_t wg) {
  int i = 0;
  while (i + 1 < b.n && wg >= b.first[i + 1]) i++;
  return i;
}

template <bool Q8>
__global__ __launch_bounds__(NT) void k_adamw(Batch b) {
#pragma clang fp contract(off)
  const int i = tensor_of(b, blockIdx.x);
  const hiertcn_adamw_tensor_t& t = b.t[i];
  const int64_t block = (int64_t)(blockIdx.x - b.first[i]) * PER_WG + (threadIdx.x >> 6);
  if (block * BLOCK >= t.numel) return;
  const Lane l = lane_of(block, t.numel, b.wide >> i & 1);
  const float gs = b.gscale_dev ? b.gscale * b.gscale_dev[0] : b.gscale;
  float p[4], g[4], m[4], v[4], s[4];
  load4<float>(t.param, l, p);
  load_grad(t, l, g);
  if constexpr (Q8) {
    int8_t qm[4];
    uint8_t qv[4];
    load4<int8_t>(t.m, l, qm);
    load4<uint8_t>(t.v, l, qv);
    const float sm = t.m_scale[block], sv = t.v_scale[block];
#pragma unroll
    for (int k = 0; k < 4; k++) m[k] = decode_m(qm[k], sm), v[k] = decode_v(qv[k], sv);
  } else {
    load4<float>(t.m, l, m);
    load4<float>(t.v, l, v);
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float gk = g[k] * gs;
    m[k] = m[k] * b.b1 + gk * b.c1;
    v[k] = v[k] * b.b2 + gk * gk * b.c2;
    s[k] = sqrtf(v[k]);
    p[k] = p[k] * b.decay[i] - b.step * (m[k] / (s[k] * b.root + b.eps));
  }
  store4<float>(t.param, l, p);
  if (t.copy) {
    uint16_t h[4];
#pragma unroll
    for (int k = 0; k < 4; k++) h[k] = t.copy_dtype == HIERTCN_BF16 ? ops_f2h(p[k], HIERTCN_BF16) : ops_f2h(p[k], HIERTCN_FP16);
    store4<uint16_t>(t.copy, l, h);
  }
  if constexpr (Q8) {
    float tm = 0.f, tv = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < l.n) {
        const float am = fabsf(m[k]);
        tm = am > tm || am != am ? am : tm;
        tv = s[k] > tv || s[k] != s[k] ? s[k] : tv;
      }
    const float sm = scale_of(wave_max(tm)), sv = scale_of(wave_max(tv));
    const float im = inverse_of(sm), iv = inverse_of(sv);
    int8_t qm[4];
    uint8_t qv[4];
    const uint32_t key = b.key + (uint32_t)t.index * 0xBB67AE85u;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t bits = mix((uint64_t)(l.base + k * l.step), key);
      const int c = encode<false>(fabsf(m[k]), im, bits & 0xffffu);
      qm[k] = (int8_t)(m[k] < 0.f ? -c : c);
      qv[k] = (uint8_t)encode<true>(s[k], iv, bits >> 16);
    }
    store4<int8_t>(t.m, l, qm);
    store4<uint8_t>(t.v, l, qv);
    if ((threadIdx.x & 63) == 0) t.m_scale[block] = sm, t.v_scale[block] = sv;
  } else {
    store4<float>(t.m, l, m);
    store4<float>(t.v, l, v);
  }
}

struct DecodeBatch {
  struct { int64_t numel; const void* m; const void* v; const float* ms; const float* vs; float* mo; float* vo; } t[MAX_TENSORS];
  uint32_t first[MAX_TENSORS + 1];
  int n;
  uint64_t wide;
};
static_assert(sizeof(DecodeBatch) <= 4096, "kernel arguments");
__global__ __launch_bounds__(NT) void k_moments(DecodeBatch b) {
  int i = 0;
  while (i + 1 < b.n && blockIdx.x >= b.first[i + 1]) i++;
  const auto& t = b.t[i];
  const int64_t block = (int64_t)(blockIdx.x - b.first[i]) * PER_WG + (threadIdx.x >> 6);
  if (block * BLOCK >= t.numel) return;
  const Lane l = lane_of(block, t.numel, b.wide >> i & 1);
  float o[4];
  if (t.mo) {
    int8_t q[4];
    load4<int8_t>(t.m, l, q);
    const float s = t.ms[block];
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] = decode_m(q[k], s);
    store4<float>(t.mo, l, o);
  }
  if (t.vo) {
    uint8_t q[4];
    load4<uint8_t>(t.v, l, q);
    const float s = t.vs[block];
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] = decode_v(q[k], s);
    store4<float>(t.vo, l, o);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------------
int check_tensor(const hiertcn_adamw_tensor_t& t, int64_t i, bool q8, bool need_param) {
  if (t.numel < 0 || t.numel > (1ll << 40)) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: %lld elements", (long long)i, (long long)t.numel);
  if (t.numel == 0) return HIERTCN_OK;
  if ((need_param && !t.param) || !t.m || !t.v || (q8 && (!t.m_scale || !t.v_scale))) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: null parameter, state or scale", (long long)i);
  if (need_param) {
    if (t.grad && !ops_dtype_ok(t.grad_dtype)) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: gradient dtype %d", (long long)i, t.grad_dtype);
    if (t.copy && t.copy_dtype != HIERTCN_BF16 && t.copy_dtype != HIERTCN_FP16) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: copy dtype %d: 1 bf16, 2 fp16", (long long)i, t.copy_dtype);
    if (!(t.weight_decay >= 0.f && t.weight_decay < 3e38f)) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: weight_decay has to be finite and not negative", (long long)i);
  }
  const int64_t blocks = (t.numel + BLOCK - 1) / BLOCK;
  const int ss = q8 ? 1 : 4;
  const OpsView v[7] = {ops_flat(need_param ? t.param : nullptr, t.numel, 4), ops_flat(t.m, t.numel, ss), ops_flat(t.v, t.numel, ss), ops_flat(need_param ? t.copy : nullptr, t.numel, 2),
                        ops_flat(q8 ? t.m_scale : nullptr, blocks, 4), ops_flat(q8 ? t.v_scale : nullptr, blocks, 4),
                        ops_flat(need_param ? t.grad : nullptr, t.numel, t.grad && need_param ? ops_size(t.grad_dtype) : 4)};
  for (int x = 0; x < 7; x++) {
    if ((uintptr_t)v[x].p % v[x].es) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: a pointer is not a multiple of its element", (long long)i);
    for (int y = 0; y < x; y++)
      if (ops_overlap(v[x], v[y])) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: two of its buffers overlap", (long long)i);
  }
  return HIERTCN_OK;
}
bool wide_of(const hiertcn_adamw_tensor_t& t, bool q8) {
  const size_t ss = q8 ? 4 : 16;
  return (uintptr_t)t.param % 16 == 0 && (uintptr_t)t.m % ss == 0 && (uintptr_t)t.v % ss == 0 && (uintptr_t)t.copy % 8 == 0 &&
         (!t.grad || (uintptr_t)t.grad % (t.grad_dtype == HIERTCN_FP32 ? 16 : 8) == 0);
}

}  // namespace

extern "C" {

int hiertcn_adamw_step(const hiertcn_adamw_tensor_t* tensors, int64_t n, const hiertcn_adamw_t* a, void* stream) {
  if (!a || n < 0 || (n > 0 && !tensors)) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  if (a->state_bits != 8 && a->state_bits != 32) return ops_fail(HIERTCN_ERR_INVALID, "state_bits %d: 8 or 32", a->state_bits);
  if (a->t < 1) return ops_fail(HIERTCN_ERR_INVALID, "t = %lld: steps count from 1", (long long)a->t);
  if (!(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1)) return ops_fail(HIERTCN_ERR_INVALID, "betas lie in [0, 1)");
  if (!(a->lr >= 0 && a->lr < 1e30 && a->eps >= 0 && a->eps < 1e30)) return ops_fail(HIERTCN_ERR_INVALID, "lr and eps have to be finite and not negative");
  if (!(a->grad_scale - a->grad_scale == 0)) return ops_fail(HIERTCN_ERR_INVALID, "grad_scale is not finite");
  if ((uintptr_t)a->grad_scale_dev % 4) return ops_fail(HIERTCN_ERR_INVALID, "grad_scale_dev is not a multiple of 4");
  const bool q8 = a->state_bits == 8;
  for (int64_t i = 0; i < n; i++)
    if (int rc = check_tensor(tensors[i], i, q8, true)) return rc;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  OPS_TRY(hipStreamIsCapturing(st, &cap));
  if (cap != hipStreamCaptureStatusNone) return ops_fail(HIERTCN_ERR_STATE, "a captured step would replay with the same t and lr: call it outside the graph");
  Batch b{};
  b.b1 = (float)a->beta1;
  b.c1 = (float)(1.0 - a->beta1);
  b.b2 = (float)a->beta2;
  b.c2 = (float)(1.0 - a->beta2);
  b.step = (float)(a->lr / (1.0 - pow(a->beta1, (double)a->t)));
  b.root = (float)(1.0 / sqrt(1.0 - pow(a->beta2, (double)a->t)));
  b.eps = (float)a->eps;
  b.gscale = (float)a->grad_scale;
  b.gscale_dev = a->grad_scale_dev;
  b.key = (uint32_t)((uint64_t)a->seed * 0x9E3779B1u + (uint64_t)a->t * 0x6A09E667u);
  for (int64_t i = 0; i < n;) {
    b.n = 0;
    b.wide = 0;
    uint64_t wgs = 0;
    for (; i < n && b.n < MAX_TENSORS; i++) {
      const hiertcn_adamw_tensor_t& t = tensors[i];
      if (t.numel == 0 || !t.grad) continue;
      const uint64_t blocks = (uint64_t)(t.numel + BLOCK - 1) / BLOCK, w = (blocks + PER_WG - 1) / PER_WG;
      if (w > 0x7fffffffull) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: too large for one launch", (long long)i);
      if (wgs + w > 0x7fffffffull) break;
      b.t[b.n] = t;
      b.decay[b.n] = (float)(1.0 - a->lr * t.weight_decay);
      b.first[b.n] = (uint32_t)wgs;
      if (wide_of(t, q8)) b.wide |= 1ull << b.n;
      b.n++;
      wgs += w;
    }
    if (!b.n) continue;
    b.first[b.n] = (uint32_t)wgs;
    if (q8) hipLaunchKernelGGL((k_adamw<true>), dim3((unsigned)wgs), dim3(NT), 0, st, b);
    else hipLaunchKernelGGL((k_adamw<false>), dim3((unsigned)wgs), dim3(NT), 0, st, b);
    OPS_TRY(hipGetLastError());
  }
  return HIERTCN_OK;
}

int hiertcn_adamw_moments(const hiertcn_adamw_tensor_t* tensors, int64_t n, float* const* m_out, float* const* v_out, void* stream) {
  if (n < 0 || (n > 0 && (!tensors || !m_out || !v_out))) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  for (int64_t i = 0; i < n; i++) {
    if (int rc = check_tensor(tensors[i], i, true, false)) return rc;
    const hiertcn_adamw_tensor_t& t = tensors[i];
    const int64_t blocks = (t.numel + BLOCK - 1) / BLOCK;
    const OpsView mo = ops_flat(m_out[i], t.numel, 4), vo = ops_flat(v_out[i], t.numel, 4);
    if ((uintptr_t)m_out[i] % 4 || (uintptr_t)v_out[i] % 4) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: a pointer is not a multiple of its element", (long long)i);
    for (const OpsView& q : {ops_flat(t.m, t.numel, 1), ops_flat(t.v, t.numel, 1), ops_flat(t.m_scale, blocks, 4), ops_flat(t.v_scale, blocks, 4)})
      if (ops_overlap(mo, q) || ops_overlap(vo, q)) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: an output overlaps a state", (long long)i);
    if (ops_overlap(mo, vo)) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: the outputs overlap", (long long)i);
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int64_t i = 0; i < n;) {
    DecodeBatch b{};
    uint64_t wgs = 0;
    for (; i < n && b.n < MAX_TENSORS; i++) {
      const hiertcn_adamw_tensor_t& t = tensors[i];
      if (t.numel == 0 || (!m_out[i] && !v_out[i])) continue;
      const uint64_t blocks = (uint64_t)(t.numel + BLOCK - 1) / BLOCK, w = (blocks + PER_WG - 1) / PER_WG;
      if (w > 0x7fffffffull) return ops_fail(HIERTCN_ERR_INVALID, "tensor %lld: too large for one launch", (long long)i);
      if (wgs + w > 0x7fffffffull) break;
      b.t[b.n] = {t.numel, t.m, t.v, t.m_scale, t.v_scale, m_out[i], v_out[i]};
      b.first[b.n] = (uint32_t)wgs;
      if ((uintptr_t)t.m % 4 == 0 && (uintptr_t)t.v % 4 == 0 && (uintptr_t)m_out[i] % 16 == 0 && (uintptr_t)v_out[i] % 16 == 0) b.wide |= 1ull << b.n;
      b.n++;
      wgs += w;
    }
    if (!b.n) continue;
    b.first[b.n] = (uint32_t)wgs;
    hipLaunchKernelGGL(k_moments, dim3((unsigned)wgs), dim3(NT), 0, st, b);
    OPS_TRY(hipGetLastError());
  }
  return HIERTCN_OK;
}

}  // extern "C"
