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
//
// 32 bits: bound by memory, 26.9 us for 5.4 M parameters (161 MB in cache, 6 TB/s).  8 bits, 155.5 M parameters with bf16 gradients and copies: 579 us for
// 2.5 GB (4.3 TB/s); by then 545 vector instructions a wave fill nine tenths of the cycles, so the instructions were what was cut (bounds of full blocks, maxima by
// lane moves, roots and quotients without the library's range handling: 725 -> 545, 706 -> 575 us).  Decoding the moments: 294 us for 1.56 GB, four blocks
// to a wave (375 us with one).
#include <math.h>

#include "ops.h"

namespace {

constexpr int NT = 256, BLOCK = 256;     // threads of a workgroup; elements of a block (one wave, four to a lane)
constexpr int PER_WG = NT / 64;          // blocks of a workgroup
constexpr int MAX_TENSORS = 40;          // of a launch: 40 descriptors fit the 4 KB of kernel arguments
constexpr uint32_t PIECE = 1u << 23;     // workgroups of a tensor in one launch, at most: a longer tensor goes in pieces

struct Batch {
  hiertcn_adamw_tensor_t t[MAX_TENSORS];
  uint32_t first[MAX_TENSORS + 1];       // first workgroup of a tensor
  int n;
  float b1, c1, b2, c2, step, root, eps, gscale;      // c = 1 - b
  float decay[MAX_TENSORS];              // 1 - lr * weight_decay
  const float* gscale_dev;
  uint32_t key;                          // of the random bits, without the tensor's share
  uint64_t wide;                         // bit i: tensor i's addresses allow four elements at a time
  uint32_t zero[MAX_TENSORS];            // where the tensor's own first workgroup would lie: first, less those of the pieces before (modulo 2^32)
};
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

// random bits of element e.  (Its high word is a block's: blocks of 256 do not cross 2^32.)
__device__ __forceinline__ uint32_t mix(uint32_t e, uint32_t key) {
  uint32_t x = e * 0x9E3779B1u + key;
  x = (x ^ (x >> 16)) * 0x3C6EF373u;
  x = (x ^ (x >> 15)) * 0x510E527Fu;
  return x ^ (x >> 16);
}

// where a lane's four elements of a block lie: neighbours where the addresses allow it, else 64 apart.  FULL: known to be all there, side by side
template <bool FULL>
struct Lane {
  int64_t base;
  int step, n;                           // element i: base + i * step; the first n exist
  __device__ __forceinline__ Lane(int64_t block, int64_t numel, bool wide) {
    const int lane = threadIdx.x & 63;
    if constexpr (FULL) wide = true;
    step = wide ? 1 : 64;
    base = block * BLOCK + (wide ? lane * 4 : lane);
    const int64_t left = numel - base;
    n = FULL ? 4 : left <= 0 ? 0 : wide ? (left < 4 ? (int)left : 4) : (int)((left + 63) / 64 < 4 ? (left + 63) / 64 : 4);
  }
};
template <typename T>
struct alignas(4 * sizeof(T)) Four { T v[4]; };
template <typename T, bool FULL>
__device__ __forceinline__ void load4(const void* p, const Lane<FULL>& l, T (&o)[4]) {
  const T* q = static_cast<const T*>(p) + l.base;
  if (FULL || (l.step == 1 && l.n == 4)) {
    const Four<T> x = *reinterpret_cast<const Four<T>*>(q);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = x.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = i < l.n ? q[i * l.step] : T(0);
  }
}
template <typename T, bool FULL>
__device__ __forceinline__ void store4(void* p, const Lane<FULL>& l, const T (&o)[4]) {
  T* q = static_cast<T*>(p) + l.base;
  if (FULL || (l.step == 1 && l.n == 4)) {
    Four<T> x;
#pragma unroll
    for (int i = 0; i < 4; i++) x.v[i] = o[i];
    ops_put<true>(q, x);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (i < l.n) q[i * l.step] = o[i];
  }
}
template <bool FULL>
__device__ __forceinline__ void load_grad(const hiertcn_adamw_tensor_t& t, const Lane<FULL>& l, float (&g)[4]) {
  if (t.grad_dtype == HIERTCN_FP32) {
    load4<float>(t.grad, l, g);
  } else {
    uint16_t h[4];
    load4<uint16_t>(t.grad, l, h);
#pragma unroll
    for (int i = 0; i < 4; i++) g[i] = t.grad_dtype == HIERTCN_BF16 ? ops_h2f(h[i], HIERTCN_BF16) : ops_h2f(h[i], HIERTCN_FP16);
  }
}
__device__ __forceinline__ float lane_of(float x, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane)); }
// the largest of the wave's magnitudes, as bits: unsigned numbers in the order of the floats they hold, NaNs above them all.  Steps of 1, 2, 4, 8 lanes inside rows
// of 16, then a row into the next and a half into the next; the last lane has it.
template <int CTRL>
__device__ __forceinline__ uint32_t max_of(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
  return x > y ? x : y;
}
__device__ __forceinline__ float wave_max(uint32_t x) {
  x = max_of<0x111>(x);
  x = max_of<0x112>(x);
  x = max_of<0x114>(x);
  x = max_of<0x118>(x);
  x = max_of<0x142>(x);
  x = max_of<0x143>(x);
  return lane_of(__builtin_bit_cast(float, x), 63);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }
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
// sqrt(v), rounded: the hardware's reciprocal root and one correction, which is the rounded root for every mantissa of both binades (all 2^24 were compared) as
// long as neither v nor the correction leaves the normal range; the library's root for zero, tiny, huge and what is no number.  Half its operations.
__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(v), x = v * y;
  float s = __builtin_fmaf(__builtin_fmaf(-x, x, v), 0.5f * y, x);
  if (__builtin_expect(__builtin_bit_cast(uint32_t, v) - 0x0d800000u >= 0x65000000u, 0)) {      // outside of 2^-100 .. 2^102
    asm volatile("");
    s = sqrtf(v);
  }
  return s;
}
// n / d to within a unit of its last place; zeros, infinities and NaNs as a division has them
__device__ __forceinline__ float quotient(float n, float d) {
  const float y = __builtin_amdgcn_rcpf(d), q = n * y;
  return __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-d, q, n), y, q), d, n);
}
// code of a magnitude: the largest a with a <= r, or the next one up with the probability that keeps the expectation
template <bool SQUARED>
__device__ __forceinline__ int encode(float mag, float inv, uint32_t bits) {
#pragma clang fp contract(off)
  constexpr float TOP = SQUARED ? 255.f : 127.f;
  float r = mag * inv;
  // q = floor(sqrt(r) TOP), at most TOP - 1.  The hardware's root is off by a unit of its last place, which matters only next to a whole number: there the
  // rounded root is taken (a lane in 2000; the empty asm keeps the compiler from taking it for all).  Cut to [1/2, TOP - 1/2] the ends are not such a place.
  float y = __builtin_amdgcn_fmed3f(__builtin_amdgcn_sqrtf(r) * TOP, 0.5f, TOP - 0.5f);
  if (__builtin_expect(fabsf(__builtin_amdgcn_fractf(y) - 0.5f) > 0.499755859375f, 0)) {
    asm volatile("");
    y = __builtin_amdgcn_fmed3f(sqrtf(r) * TOP, 0.5f, TOP - 0.5f);
  }
  const float q = floorf(y);
  float a = q * (1.f / TOP), b = (q + 1.f) * (1.f / TOP);
  a = a * a;
  b = b * b;
  if (SQUARED) {
    a = a * a;
    b = b * b;
    r = r * r;
  }
  const float u = (float)bits * 1.52587890625e-5f;
  const int code = (int)q + (r - a > u * (b - a) ? 1 : 0);
  return SQUARED && mag > 0.f && inv > 0.f && code < 1 ? 1 : code;
}
__device__ __forceinline__ float scale_of(float largest) { return largest < 7.888609052210118e-31f ? 0.f : largest; }      // 2^-100
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.f ? 1.f / scale : 0.f; }

template <typename B>
__device__ __forceinline__ int tensor_of(const B& b, uint32_t wg) {
  int i = 0;
  while (i + 1 < b.n && wg >= b.first[i + 1]) i++;
  return i;
}

template <bool Q8, bool FULL>
__device__ __forceinline__ void update(const Batch& b, const hiertcn_adamw_tensor_t& t, int64_t block, bool wide, float decay) {
#pragma clang fp contract(off)
  const Lane<FULL> l(block, t.numel, wide);
  const float gs = b.gscale_dev ? b.gscale * b.gscale_dev[0] : b.gscale;
  float p[4], g[4], m[4], v[4], s[4];
  if constexpr (Q8) {
    int8_t qm[4];
    uint8_t qv[4];
    load4<int8_t>(t.m, l, qm);
    load4<uint8_t>(t.v, l, qv);
    const float sm = t.m_scale[block], sv = t.v_scale[block];
    load4<float>(t.param, l, p);
    load_grad(t, l, g);
#pragma unroll
    for (int k = 0; k < 4; k++) m[k] = decode_m(qm[k], sm), v[k] = decode_v(qv[k], sv);
  } else {
    load4<float>(t.m, l, m);
    load4<float>(t.v, l, v);
    load4<float>(t.param, l, p);
    load_grad(t, l, g);
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float gk = g[k] * gs;
    m[k] = m[k] * b.b1 + gk * b.c1;
    v[k] = v[k] * b.b2 + gk * gk * b.c2;
    s[k] = root_of(v[k]);
    p[k] = p[k] * decay - b.step * quotient(m[k], s[k] * b.root + b.eps);
  }
  store4<float>(t.param, l, p);
  if (t.copy) {
    uint16_t h[4];
#pragma unroll
    for (int k = 0; k < 4; k++) h[k] = t.copy_dtype == HIERTCN_BF16 ? ops_f2h(p[k], HIERTCN_BF16) : ops_f2h(p[k], HIERTCN_FP16);
    store4<uint16_t>(t.copy, l, h);
  }
  if constexpr (Q8) {
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (k < l.n) {
        tm = tm > magnitude(m[k]) ? tm : magnitude(m[k]);
        tv = tv > magnitude(s[k]) ? tv : magnitude(s[k]);
      }
    const float sm = scale_of(wave_max(tm)), sv = scale_of(wave_max(tv));
    const float inv = inverse_of(threadIdx.x & 1 ? sv : sm);                                    // one division for both
    const float im = lane_of(inv, 0), iv = lane_of(inv, 1);
    int8_t qm[4];
    uint8_t qv[4];
    const uint32_t key = b.key + (uint32_t)t.index * 0xBB67AE85u + (uint32_t)((uint64_t)(block * BLOCK) >> 32) * 0x1F83D9ABu;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t bits = mix((uint32_t)(l.base + k * l.step), key);
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

// the wave's first block of its tensor, of EACH.  false: behind its end
template <int EACH, typename B>
__device__ __forceinline__ bool block_here(const B& b, int i, int64_t& block) {
  block = ((int64_t)(blockIdx.x - b.zero[i]) * PER_WG + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * EACH;
  return block * BLOCK < b.t[i].numel;
}
template <bool Q8>
__global__ __launch_bounds__(NT) void k_adamw(Batch b) {
  const int i = tensor_of(b, blockIdx.x);
  int64_t block;
  if (!block_here<1>(b, i, block)) return;
  const bool wide = b.wide >> i & 1;
  if (wide && (block + 1) * BLOCK <= b.t[i].numel) update<Q8, true>(b, b.t[i], block, wide, b.decay[i]);
  else update<Q8, false>(b, b.t[i], block, wide, b.decay[i]);
}

struct DecodeBatch {
  struct { int64_t numel; const void* m; const void* v; const float* ms; const float* vs; float* mo; float* vo; } t[MAX_TENSORS];
  uint32_t first[MAX_TENSORS + 1];
  int n;
  uint64_t wide;
  uint32_t zero[MAX_TENSORS];
};
static_assert(sizeof(DecodeBatch) <= 4096, "kernel arguments");
// a wave decodes WAVE_BLOCKS blocks of a tensor, all loads first
constexpr int WAVE_BLOCKS = 4;
template <bool FULL, typename T>
__device__ __forceinline__ void decode_blocks(const T& t, int64_t block, bool wide) {
  int8_t qm[WAVE_BLOCKS][4];
  uint8_t qv[WAVE_BLOCKS][4];
  float sm[WAVE_BLOCKS], sv[WAVE_BLOCKS], o[4];
#pragma unroll
  for (int j = 0; j < WAVE_BLOCKS; j++) {
    const Lane<FULL> l(block + j, t.numel, wide);
    const bool here = FULL || (block + j) * BLOCK < t.numel;
    if (t.mo) load4<int8_t>(t.m, l, qm[j]), sm[j] = here ? t.ms[block + j] : 0.f;
    if (t.vo) load4<uint8_t>(t.v, l, qv[j]), sv[j] = here ? t.vs[block + j] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < WAVE_BLOCKS; j++) {
    const Lane<FULL> l(block + j, t.numel, wide);
    if (t.mo) {
#pragma unroll
      for (int k = 0; k < 4; k++) o[k] = decode_m(qm[j][k], sm[j]);
      store4<float>(t.mo, l, o);
    }
    if (t.vo) {
#pragma unroll
      for (int k = 0; k < 4; k++) o[k] = decode_v(qv[j][k], sv[j]);
      store4<float>(t.vo, l, o);
    }
  }
}
__global__ __launch_bounds__(NT) void k_moments(DecodeBatch b) {
  const int i = tensor_of(b, blockIdx.x);
  int64_t block;
  if (!block_here<WAVE_BLOCKS>(b, i, block)) return;
  const bool wide = b.wide >> i & 1;
  if (wide && (block + WAVE_BLOCKS) * BLOCK <= b.t[i].numel) decode_blocks<true>(b.t[i], block, wide);
  else decode_blocks<false>(b.t[i], block, wide);
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
// The launches of a call, one after the other: which pieces of which tensors go into the next one, `each` blocks to a wave.  All that a call can refuse is
// refused before the first of them.
struct Walk {
  const hiertcn_adamw_tensor_t* t;
  int64_t n, i, piece;
  int each;
  int64_t tensor[MAX_TENSORS];           // the launch at hand
  uint32_t first[MAX_TENSORS + 1];
  uint8_t which[MAX_TENSORS];
  int count;
  Walk(const hiertcn_adamw_tensor_t* t, int64_t n, int each) : t(t), n(n), i(0), piece(0), each(each), count(0) {}
  // works(i): whether tensor i takes part.  -> its number of workgroups, 0 behind the last
  template <typename F>
  uint32_t next(F works) {
    int64_t wgs = 0;
    for (count = 0; i < n && count < MAX_TENSORS;) {
      if (t[i].numel == 0 || !works(i)) {
        i++;
        continue;
      }
      const int64_t span = (int64_t)BLOCK * PER_WG * each, all = (t[i].numel + span - 1) / span, left = all - piece * PIECE, w = left < PIECE ? left : PIECE;
      if (wgs + w > ops_most_groups(NT)) break;
      tensor[count] = i;
      first[count] = (uint32_t)wgs;
      which[count++] = (uint8_t)piece;
      wgs += w;
      if (w < left) piece++;
      else i++, piece = 0;
    }
    first[count] = (uint32_t)wgs;
    return (uint32_t)wgs;
  }
};
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
  Walk walk(tensors, n, 1);
  while (const uint32_t wgs = walk.next([&](int64_t i) { return tensors[i].grad != nullptr; })) {
    b.n = walk.count;
    b.wide = 0;
    for (int k = 0; k < b.n; k++) {
      const hiertcn_adamw_tensor_t& t = tensors[walk.tensor[k]];
      b.t[k] = t;
      b.decay[k] = (float)(1.0 - a->lr * t.weight_decay);
      b.first[k] = walk.first[k];
      b.zero[k] = walk.first[k] - walk.which[k] * PIECE;
      if (wide_of(t, q8)) b.wide |= 1ull << k;
    }
    b.first[b.n] = wgs;
    if (q8) hipLaunchKernelGGL((k_adamw<true>), dim3(wgs), dim3(NT), 0, st, b);
    else hipLaunchKernelGGL((k_adamw<false>), dim3(wgs), dim3(NT), 0, st, b);
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
  Walk walk(tensors, n, WAVE_BLOCKS);
  while (const uint32_t wgs = walk.next([&](int64_t i) { return m_out[i] || v_out[i]; })) {
    DecodeBatch b{};
    b.n = walk.count;
    for (int k = 0; k < b.n; k++) {
      const int64_t i = walk.tensor[k];
      const hiertcn_adamw_tensor_t& t = tensors[i];
      b.t[k] = {t.numel, t.m, t.v, t.m_scale, t.v_scale, m_out[i], v_out[i]};
      b.first[k] = walk.first[k];
      b.zero[k] = walk.first[k] - walk.which[k] * PIECE;
      if ((uintptr_t)t.m % 4 == 0 && (uintptr_t)t.v % 4 == 0 && (uintptr_t)m_out[i] % 16 == 0 && (uintptr_t)v_out[i] % 16 == 0) b.wide |= 1ull << k;
    }
    b.first[b.n] = wgs;
    hipLaunchKernelGGL(k_moments, dim3(wgs), dim3(NT), 0, st, b);
    OPS_TRY(hipGetLastError());
  }
  return HIERTCN_OK;
}

#ifdef HIERTCN_TEST_HOOKS       // (the launches of a call on tensors of these sizes, for a test on the host: rows of launch, tensor, piece, first workgroup, the launch's workgroups)
int64_t hiertcn_test_adamw_walk(const int64_t* numel, int64_t n, int each, int64_t* out, int64_t room) {
  hiertcn_adamw_tensor_t t[256] = {};
  if (n > 256) return -1;
  for (int64_t i = 0; i < n; i++) t[i].numel = numel[i];
  Walk walk(t, n, each);
  int64_t rows = 0, launch = 0;
  for (; const uint32_t wgs = walk.next([](int64_t) { return true; }); launch++)
    for (int k = 0; k < walk.count; k++, rows++) {
      if (rows == room) return -1;
      const int64_t row[5] = {launch, walk.tensor[k], walk.which[k], walk.first[k], wgs};
      for (int x = 0; x < 5; x++) out[5 * rows + x] = row[x];
    }
  return rows;
}
int hiertcn_test_adamw_sizes(int64_t out[4]) {
  out[0] = PIECE, out[1] = BLOCK * PER_WG, out[2] = MAX_TENSORS, out[3] = NT;
  return WAVE_BLOCKS;
}
#endif

}  // extern "C"
