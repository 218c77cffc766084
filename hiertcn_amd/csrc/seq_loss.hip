// Losses on the log-probabilities of answers, with their gradients to the logits (include/hiertcn_ops.h).
//
// Every loss here is a function of logp = z_y - m - ln s per row (m the row's largest logit, s = sum exp(z - m)), so its gradient to a row is
//   dz_j = c (  [j = y] - exp(z_j - m) / s ),   c = d loss / d logp,
// and a loss differs from another only in how c comes from the logp's.  Three launches:
//   k_part    one pass over the logits: (m, s) of every part of every row, running maximum and sum
//   k_pairs / k_policy / k_logp   joins a row's parts, forms logp, the loss and c
//   k_dlogits one pass over the logits: dz  (its last workgroup adds up the loss)
// Masked rows are not read: their gradient rows are written as zeros.  All sums run in a fixed order.
#include <math.h>

#include "ops.h"

namespace {

constexpr int NT = 256;                 // threads of a workgroup
constexpr int MAX_PARTS = 64;

struct RowsP {
  hiertcn_rows_t a;
  int64_t R;
  int parts;
  int64_t chunk;                        // vectors of a part
  float2* part;                         // [R][parts] (m, s)
  float2* stat;                         // [R] (m, 1 / s)
  float* coef;                          // [R] d (grad_scale * loss) / d logp
  float* term;                          // [3][R] policy: weighted loss, kl, clipped per row
  int32_t* count;                       // [n] policy: answers of a sequence
};

__device__ __forceinline__ bool answered(const hiertcn_rows_t& a, int64_t r, int32_t& y) {
  y = a.ids[r];
  return y > 0 && y < a.V;
}

// (m, s) of two runs as one.  m = -inf: nothing in it (s is 0, or NaN and stays NaN).
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = ref_of(top);
  s = s * ops_exp(m - ref) + s2 * ops_exp(m2 - ref);
  m = top;
}
__device__ __forceinline__ void wave_join(float& m, float& s) {
#pragma unroll
  for (int d = 32; d; d >>= 1) join(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
}

// the part of a row as [head] vectors [tail]: head elements up to the first address that a vector may be loaded from
template <int DT, int VEC>
struct Span {
  int64_t head, nvec, v0, v1;           // v0 .. v1: this part's vectors; element of vector v: head + v * VEC
  int64_t tail;                         // first element behind the vectors
  __device__ Span(const void* row, int64_t V, int64_t chunk, int part) {
    constexpr int ES = DT == HIERTCN_FP32 ? 4 : 2;
    head = VEC == 1 ? 0 : (int64_t)((16 - ((uintptr_t)row & 15)) & 15) / ES;
    if (head > V) head = V;
    nvec = (V - head) / VEC;
    tail = head + nvec * VEC;
    v0 = part * chunk;
    v1 = v0 + chunk < nvec ? v0 + chunk : nvec;
  }
};
template <int DT>
__device__ __forceinline__ const void* row_of(const void* p, int64_t off) {
  return DT == HIERTCN_FP32 ? (const void*)(static_cast<const float*>(p) + off) : (const void*)(static_cast<const uint16_t*>(p) + off);
}

template <int DT, int VEC>
__global__ __launch_bounds__(NT) void k_part(RowsP p) {
  constexpr int U = 4;
  const hiertcn_rows_t& a = p.a;
  if ((int64_t)blockIdx.x >= p.R * p.parts) {                  // policy: the answers of a sequence
    const int64_t q = blockIdx.x - p.R * p.parts;
    int c = 0;
    for (int64_t t = threadIdx.x; t < a.T; t += NT) {
      int32_t y;
      c += answered(a, q * a.T + t, y);
    }
    __shared__ int cs[NT / 64];
#pragma unroll
    for (int d = 32; d; d >>= 1) c += __shfl_xor(c, d);
    if ((threadIdx.x & 63) == 0) cs[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) p.count[q] = cs[0] + cs[1] + cs[2] + cs[3];
    return;
  }
  const int64_t r = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x % p.parts);
  int32_t y;
  if (!answered(a, r, y)) return;
  const void* row = row_of<DT>(a.logits, r * a.ld);
  const Span<DT, VEC> sp(row, a.V, p.chunk, part);
  float m = -INFINITY, s = 0.f;
  for (int64_t v = sp.v0 + threadIdx.x; v < sp.v1; v += NT * U) {
    float z[U][VEC], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (v + u * NT < sp.v1) ops_ld<DT, VEC>(row, sp.head + (v + u * NT) * VEC, z[u]);
      else
#pragma unroll
        for (int i = 0; i < VEC; i++) z[u][i] = -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < VEC; i++) top = fmaxf(top, z[u][i]);
    top = fmaxf(top, m);
    const float ref = ref_of(top);
    s *= ops_exp(m - ref);
    m = top;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int i = 0; i < VEC; i++) s += ops_exp(z[u][i] - ref);
  }
  // the elements in front of and behind the vectors
  int64_t e = -1;
  if (part == 0 && threadIdx.x < sp.head) e = threadIdx.x;
  if (part == p.parts - 1 && threadIdx.x >= 32 && sp.tail + (threadIdx.x - 32) < a.V) {
    e = sp.tail + (threadIdx.x - 32);
  }
  if (e >= 0) {
    float z[1];
    ops_ld<DT, 1>(row, e, z);
    join(m, s, z[0], z[0] == -INFINITY ? 0.f : ops_exp(z[0] - z[0]));
  }
  __shared__ float ms[NT / 64], ss[NT / 64];
  wave_join(m, s);
  if ((threadIdx.x & 63) == 0) ms[threadIdx.x >> 6] = m, ss[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < NT / 64; w++) join(m, s, ms[w], ss[w]);
    p.part[r * p.parts + part] = make_float2(m, s);
  }
}

__device__ __forceinline__ float logit(const hiertcn_rows_t& a, int64_t off) {
  return a.dtype == HIERTCN_FP32 ? static_cast<const float*>(a.logits)[off] : ops_h2f(static_cast<const uint16_t*>(a.logits)[off], a.dtype);
}

// logp of a row from its parts; (m, 1 / s) kept for the gradient.  false: masked, or nothing but -inf
__device__ bool finish_row(const RowsP& p, int64_t r, float& logp) {
  const hiertcn_rows_t& a = p.a;
  int32_t y;
  logp = 0.f;
  if (!answered(a, r, y)) return false;
  float m = -INFINITY, s = 0.f;
  for (int q = 0; q < p.parts; q++) {
    const float2 x = p.part[r * p.parts + q];
    join(m, s, x.x, x.y);
  }
  p.stat[r] = make_float2(m, 1.f / s);
  if (m == -INFINITY && s == 0.f) return false;
  logp = (logit(a, r * a.ld + y) - ref_of(m)) - logf(s);
  return true;
}

__global__ __launch_bounds__(NT) void k_logp(RowsP p) {
  const int64_t r = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (r >= p.R) return;
  float lp;
  finish_row(p, r, lp);
  p.a.logp[r] = lp;
}

__device__ double block_sum(double x) {
  __shared__ double t[NT / 64];
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) t[threadIdx.x >> 6] = x;
  __syncthreads();
  return t[0] + t[1] + t[2] + t[3];
}
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// a workgroup a pair: both sums, the loss, the slope d loss / d s
__global__ __launch_bounds__(NT) void k_pairs(RowsP p, hiertcn_preference_t q) {
  const hiertcn_rows_t& a = p.a;
  const int64_t P = a.n / 2;
  double s[2];
  double cnt[2];
  for (int side = 0; side < 2; side++) {
    const int64_t seq = blockIdx.x + side * P;
    double sum = 0.0, c = 0.0;
    for (int64_t t = threadIdx.x; t < a.T; t += NT) {
      const int64_t r = seq * a.T + t;
      float lp;
      const bool live = finish_row(p, r, lp);
      a.logp[r] = lp;
      int32_t y;
      c += answered(a, r, y);
      p.coef[r] = live ? 1.f : 0.f;
      sum += lp;
    }
    sum = block_sum(sum);
    cnt[side] = block_sum(c);
    s[side] = q.average ? (cnt[side] > 0 ? sum / cnt[side] : 0.0) : sum;
  }
  const double beta = q.beta, eps = q.smoothing, D = (s[0] - q.ref[blockIdx.x]) - (s[1] - q.ref[blockIdx.x + P]);
  double loss, slope;
  if (q.kind == 0) {
    loss = (1.0 - eps) * softplus(-beta * D) + (eps > 0.0 ? eps * softplus(beta * D) : 0.0);
    slope = beta * (1.0 / (1.0 + exp(-beta * D)) - (1.0 - eps));
  } else if (q.kind == 1) {
    loss = 1.0 - beta * D > 0.0 ? 1.0 - beta * D : (D != D ? D : 0.0);
    slope = 1.0 - beta * D > 0.0 ? -beta : (D != D ? D : 0.0);
  } else {
    const double off = D - 0.5 / beta;
    loss = off * off;
    slope = 2.0 * off;
  }
  if (threadIdx.x == 0) {
    q.pair_loss[blockIdx.x] = (float)loss;
    q.margin[blockIdx.x] = (float)D;
    q.seq_logp[blockIdx.x] = (float)s[0];
    q.seq_logp[blockIdx.x + P] = (float)s[1];
  }
  for (int side = 0; side < 2; side++) {
    const int64_t seq = blockIdx.x + side * P;
    const double c = (side ? -slope : slope) / (double)P * a.grad_scale / (q.average ? (cnt[side] > 0 ? cnt[side] : 1.0) : 1.0);
    for (int64_t t = threadIdx.x; t < a.T; t += NT) {        // (this thread's own rows of the loop above)
      const int64_t r = seq * a.T + t;
      p.coef[r] = p.coef[r] != 0.f ? (float)c : 0.f;
    }
  }
}

// a thread a row
__global__ __launch_bounds__(NT) void k_policy(RowsP p, hiertcn_policy_t q) {
  const hiertcn_rows_t& a = p.a;
  double total = 0.0;                    // sequences with answers, or answers
  for (int64_t i = threadIdx.x; i < a.n; i += NT) total += q.mean == 0 ? (p.count[i] > 0 ? 1.0 : 0.0) : (double)p.count[i];
  total = block_sum(total);
  const int64_t r = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (r >= p.R) return;
  const int64_t b = r / a.T, t = r % a.T;
  float lp;
  const bool live = finish_row(p, r, lp);
  a.logp[r] = lp;
  float loss = 0.f, kl = 0.f, cut = 0.f, c = 0.f;
  if (live) {
    const float weight = (float)(1.0 / (q.mean == 0 ? total * p.count[b] : total));
    const float A = q.advantage[b * q.adv_sn + t * q.adv_st];
    const float ratio = expf(lp - q.old_logp[r]);
    const float lo = 1.f - q.clip_low, hi = 1.f + q.clip_high;
    const float held = ratio < lo ? lo : ratio > hi ? hi : ratio;
    const float none = lp != lp ? lp : 0.f;       // 0, or the NaN of the row
    const float x = A == 0.f ? none : ratio * A, y = A == 0.f ? none : held * A;
    const bool clipped = x > y;
    loss = clipped ? -y : -x;
    cut = clipped ? weight : 0.f;
    c = clipped ? none : -x;
    if (q.ref_logp) {
      const float gap = q.ref_logp[r] - lp, e = expf(gap);
      kl = e == INFINITY ? e : (e - gap) - 1.f;
      if (fabsf(gap) < 0.25f)            // e^gap - gap - 1 loses its digits there: the series
        kl = gap * gap * fmaf(gap, fmaf(gap, fmaf(gap, fmaf(gap, fmaf(gap, 1.f / 5040.f, 1.f / 720.f), 1.f / 120.f), 1.f / 24.f), 1.f / 6.f), 0.5f);
      loss += q.kl_coef * kl;
      c += q.kl_coef * -expm1f(gap);
    }
    loss *= weight;
    kl *= weight;
    c *= weight * a.grad_scale;
  }
  p.coef[r] = c;
  p.term[r] = loss;
  p.term[p.R + r] = kl;
  p.term[2 * p.R + r] = cut;
}

// out[k] = scale * sum of src[k * n ..], one workgroup
struct Sums { const float* src; int64_t n; float scale; float* out[3]; };
__device__ void add_up(const Sums& q) {
  for (int k = 0; k < 3; k++) {
    if (!q.out[k]) continue;
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < q.n; i += NT) x += q.src[k * q.n + i];
    x = block_sum(x);
    if (threadIdx.x == 0) q.out[k][0] = (float)(x * q.scale);
  }
}
__global__ __launch_bounds__(NT) void k_sums(Sums q) { add_up(q); }

template <int DT, int VEC>
__global__ __launch_bounds__(NT) void k_dlogits(RowsP p, Sums q) {
  constexpr int U = 4;
  const hiertcn_rows_t& a = p.a;
  if ((int64_t)blockIdx.x >= p.R * p.parts) {
    add_up(q);
    return;
  }
  const int64_t r = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x % p.parts);
  const void* row = row_of<DT>(a.logits, r * a.ld);
  void* out = const_cast<void*>(row_of<DT>(a.dlogits, r * a.dld));
  const Span<DT, VEC> sp(out, a.V, p.chunk, part);
  const float c = p.coef[r];
  int64_t e = -1;
  if (part == 0 && threadIdx.x < sp.head) e = threadIdx.x;
  if (part == p.parts - 1 && threadIdx.x >= 32 && sp.tail + (threadIdx.x - 32) < a.V) e = sp.tail + (threadIdx.x - 32);
  if (c == 0.f) {
    const float zero[VEC] = {};
    for (int64_t v = sp.v0 + threadIdx.x; v < sp.v1; v += NT) ops_st<DT, VEC>(out, sp.head + v * VEC, zero);
    const float z1[1] = {0.f};
    if (e >= 0) ops_st<DT, 1>(out, e, z1);
    return;
  }
  const int32_t y = a.ids[r];
  const float2 st = p.stat[r];
  const float ref = ref_of(st.x), g = -c * st.y;
  for (int64_t v = sp.v0 + threadIdx.x; v < sp.v1; v += NT * U) {
    float z[U][VEC];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (v + u * NT < sp.v1) ops_ld<DT, VEC>(row, sp.head + (v + u * NT) * VEC, z[u]);
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (v + u * NT >= sp.v1) break;
      const int64_t at = sp.head + (v + u * NT) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        z[u][i] = g * ops_exp(z[u][i] - ref);
        if (at + i == y) z[u][i] += c;
      }
      ops_st<DT, VEC>(out, at, z[u]);
    }
  }
  if (e >= 0) {
    float z[1];
    ops_ld<DT, 1>(row, e, z);
    z[0] = g * ops_exp(z[0] - ref);
    if (e == y) z[0] += c;
    ops_st<DT, 1>(out, e, z);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------------
size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
int64_t chunk_of(int64_t V, int vec) {         // vectors of a part: 8192 elements, more where that would make over MAX_PARTS parts
  int64_t elems = 8192;
  if ((V + elems - 1) / elems > MAX_PARTS) elems = (V + MAX_PARTS - 1) / MAX_PARTS;
  return (elems + vec - 1) / vec;
}
int parts_of(int64_t V, int vec) {
  const int64_t c = chunk_of(V, vec), nvec = V / vec;
  return (int)(nvec <= c ? 1 : (nvec + c - 1) / c);
}
size_t workspace_of(int64_t n, int64_t T, int64_t V, RowsP* p) {
  const size_t R = (size_t)(n * T);
  int most = 1;
  for (int vec : {1, 4, 8})
    if (parts_of(V, vec) > most) most = parts_of(V, vec);
  const size_t sizes[5] = {align_up(R * most * 8), align_up(R * 8), align_up(R * 4), align_up(R * 12), align_up((size_t)n * 4)};
  if (p) {
    char* w = static_cast<char*>(p->a.workspace);
    p->part = reinterpret_cast<float2*>(w);
    p->stat = reinterpret_cast<float2*>(w += sizes[0]);
    p->coef = reinterpret_cast<float*>(w += sizes[1]);
    p->term = reinterpret_cast<float*>(w += sizes[2]);
    p->count = reinterpret_cast<int32_t*>(w += sizes[3]);
  }
  return sizes[0] + sizes[1] + sizes[2] + sizes[3] + sizes[4];
}

// the checks that all entries share; sets up p
int prepare(const hiertcn_rows_t* in, bool grad, RowsP& p, int& vec) {
  if (!in) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  p.a = *in;
  hiertcn_rows_t& a = p.a;
  if (!grad) a.dlogits = nullptr;
  if (a.n < 1 || a.T < 1 || a.V < 1) return ops_fail(HIERTCN_ERR_INVALID, "n, T and V are at least 1 (%lld, %lld, %lld)", (long long)a.n, (long long)a.T, (long long)a.V);
  if (a.n > (1ll << 31) || a.T > (1ll << 31) || a.n * a.T > (1ll << 31) || a.V > 0x7fffffff) return ops_fail(HIERTCN_ERR_INVALID, "n * T is at most 2^31, V below 2^31");
  if (!ops_dtype_ok(a.dtype)) return ops_fail(HIERTCN_ERR_INVALID, "dtype %d: 0 fp32, 1 bf16, 2 fp16", a.dtype);
  if (!a.logits || !a.ids || !a.logp) return ops_fail(HIERTCN_ERR_INVALID, "null logits, ids or logp");
  p.R = a.n * a.T;
  if (p.R == 1) a.ld = a.V, a.dld = a.dlogits ? a.V : 0;
  if (a.ld < a.V || a.ld > (1ll << 40) || (a.dlogits && (a.dld < a.V || a.dld > (1ll << 40)))) return ops_fail(HIERTCN_ERR_INVALID, "a row stride is smaller than V");
  const int es = ops_size(a.dtype);
  if ((uintptr_t)a.logits % es || (uintptr_t)a.dlogits % es || (uintptr_t)a.ids % 4 || (uintptr_t)a.logp % 4)
    return ops_fail(HIERTCN_ERR_INVALID, "a pointer is not a multiple of its element");
  if (!(a.grad_scale - a.grad_scale == 0.f)) return ops_fail(HIERTCN_ERR_INVALID, "grad_scale is not finite");
  const size_t need = workspace_of(a.n, a.T, a.V, nullptr);
  if (!a.workspace || a.workspace_bytes < need || (uintptr_t)a.workspace % 16)
    return ops_fail(HIERTCN_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", need, a.workspace ? a.workspace_bytes : (size_t)0);
  const OpsView z{static_cast<const char*>(a.logits), 1, p.R, a.V, 0, a.ld, es}, d{static_cast<const char*>(a.dlogits), 1, p.R, a.V, 0, a.dld, es};
  const OpsView ids = ops_flat(a.ids, p.R, 4), lp = ops_flat(a.logp, p.R, 4), ws = ops_flat(a.workspace, (int64_t)a.workspace_bytes, 1);
  if (!(a.dlogits == a.logits && a.dld == a.ld) && ops_overlap(z, d)) return ops_fail(HIERTCN_ERR_INVALID, "dlogits overlaps logits without being the same buffer");
  for (const OpsView* o : {&lp, &ws})
    if (ops_overlap(*o, z) || ops_overlap(*o, ids) || ops_overlap(*o, d)) return ops_fail(HIERTCN_ERR_INVALID, "logp or the workspace overlaps another operand");
  if (ops_overlap(lp, ws) || ops_overlap(ids, d)) return ops_fail(HIERTCN_ERR_INVALID, "logp or the workspace overlaps another operand");
  // 16 bytes at a time wherever the two passes' rows are 16-byte aligned alike; else one element
  vec = 16 / es;
  if (a.dlogits && (((uintptr_t)a.logits - (uintptr_t)a.dlogits) % 16 || (a.ld - a.dld) % vec)) vec = 1;
  p.parts = parts_of(a.V, vec);
  p.chunk = chunk_of(a.V, vec);
  workspace_of(a.n, a.T, a.V, &p);
  if (p.R * p.parts + a.n > 0x7fffffffll) return ops_fail(HIERTCN_ERR_INVALID, "n * T * V is too large for one launch");
  return HIERTCN_OK;
}

#define ROWS_GO(kernel, blocks, ...)                                                                                                           \
  do {                                                                                                                                         \
    const dim3 g_((unsigned)(blocks)), b_(NT);                                                                                                 \
    if (p.a.dtype == HIERTCN_FP32 && vec == 1) hipLaunchKernelGGL((kernel<HIERTCN_FP32, 1>), g_, b_, 0, st, __VA_ARGS__);                       \
    else if (p.a.dtype == HIERTCN_FP32) hipLaunchKernelGGL((kernel<HIERTCN_FP32, 4>), g_, b_, 0, st, __VA_ARGS__);                              \
    else if (p.a.dtype == HIERTCN_BF16 && vec == 1) hipLaunchKernelGGL((kernel<HIERTCN_BF16, 1>), g_, b_, 0, st, __VA_ARGS__);                  \
    else if (p.a.dtype == HIERTCN_BF16) hipLaunchKernelGGL((kernel<HIERTCN_BF16, 8>), g_, b_, 0, st, __VA_ARGS__);                              \
    else if (vec == 1) hipLaunchKernelGGL((kernel<HIERTCN_FP16, 1>), g_, b_, 0, st, __VA_ARGS__);                                               \
    else hipLaunchKernelGGL((kernel<HIERTCN_FP16, 8>), g_, b_, 0, st, __VA_ARGS__);                                                             \
    OPS_TRY(hipGetLastError());                                                                                                                 \
  } while (0)

int check_out(const RowsP& p, const void* q, int64_t n, const char* name) {
  if (!q || (uintptr_t)q % 4) return ops_fail(HIERTCN_ERR_INVALID, "%s: null or not a multiple of 4", name);
  const hiertcn_rows_t& a = p.a;
  const OpsView v = ops_flat(q, n, 4);
  const int es = ops_size(a.dtype);
  for (const OpsView& o : {OpsView{static_cast<const char*>(a.logits), 1, p.R, a.V, 0, a.ld, es}, OpsView{static_cast<const char*>(a.dlogits), 1, p.R, a.V, 0, a.dld, es},
                           ops_flat(a.ids, p.R, 4), ops_flat(a.logp, p.R, 4), ops_flat(a.workspace, (int64_t)a.workspace_bytes, 1)})
    if (ops_overlap(v, o)) return ops_fail(HIERTCN_ERR_INVALID, "%s overlaps another operand", name);
  return HIERTCN_OK;
}

int finish(const RowsP& p, int vec, const Sums& s, hipStream_t st) {
  if (p.a.dlogits) {
    ROWS_GO(k_dlogits, p.R * p.parts + 1, p, s);
  } else {
    hipLaunchKernelGGL(k_sums, dim3(1), dim3(NT), 0, st, s);
    OPS_TRY(hipGetLastError());
  }
  return HIERTCN_OK;
}

}  // namespace

extern "C" {

size_t hiertcn_rows_workspace_bytes(int64_t n, int64_t T, int64_t V) {
  return n < 1 || T < 1 || V < 1 || n > (1ll << 31) || T > (1ll << 31) || n * T > (1ll << 31) || V > 0x7fffffff ? 0 : workspace_of(n, T, V, nullptr);
}

int hiertcn_sequence_logp(const hiertcn_rows_t* r, void* stream) {
  RowsP p{};
  int vec;
  if (int rc = prepare(r, false, p, vec)) return rc;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  ROWS_GO(k_part, p.R * p.parts, p);
  hipLaunchKernelGGL(k_logp, dim3((unsigned)((p.R + NT - 1) / NT)), dim3(NT), 0, st, p);
  OPS_TRY(hipGetLastError());
  return HIERTCN_OK;
}

int hiertcn_preference_loss(const hiertcn_rows_t* r, const hiertcn_preference_t* q, void* stream) {
  RowsP p{};
  int vec;
  if (!q) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  if (int rc = prepare(r, true, p, vec)) return rc;
  const int64_t n = p.a.n, P = n / 2;
  if (n % 2) return ops_fail(HIERTCN_ERR_INVALID, "%lld sequences: pairs are wanted", (long long)n);
  if (q->kind < 0 || q->kind > 2) return ops_fail(HIERTCN_ERR_INVALID, "kind %d: 0 sigmoid, 1 hinge, 2 squared", q->kind);
  if (!(q->beta > 0.f) || q->beta > 3e38f) return ops_fail(HIERTCN_ERR_INVALID, "beta has to be positive and finite");
  if (!(q->smoothing >= 0.f && q->smoothing < 0.5f)) return ops_fail(HIERTCN_ERR_INVALID, "smoothing lies in [0, 0.5)");
  if (q->kind != 0 && q->smoothing != 0.f) return ops_fail(HIERTCN_ERR_INVALID, "smoothing belongs to kind 0");
  if (!q->ref || (uintptr_t)q->ref % 4) return ops_fail(HIERTCN_ERR_INVALID, "ref: null or not a multiple of 4");
  const struct { float* q; int64_t n; const char* name; } outs[4] = {{q->loss, 1, "loss"}, {q->pair_loss, P, "pair_loss"}, {q->margin, P, "margin"}, {q->seq_logp, n, "seq_logp"}};
  for (int i = 0; i < 4; i++) {
    if (int rc = check_out(p, outs[i].q, outs[i].n, outs[i].name)) return rc;
    if (ops_overlap(ops_flat(outs[i].q, outs[i].n, 4), ops_flat(q->ref, n, 4))) return ops_fail(HIERTCN_ERR_INVALID, "%s overlaps ref", outs[i].name);
    for (int j = 0; j < i; j++)
      if (ops_overlap(ops_flat(outs[i].q, outs[i].n, 4), ops_flat(outs[j].q, outs[j].n, 4))) return ops_fail(HIERTCN_ERR_INVALID, "%s overlaps %s", outs[i].name, outs[j].name);
  }
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  ROWS_GO(k_part, p.R * p.parts, p);
  hipLaunchKernelGGL(k_pairs, dim3((unsigned)P), dim3(NT), 0, st, p, *q);
  OPS_TRY(hipGetLastError());
  return finish(p, vec, Sums{q->pair_loss, P, 1.f / (float)P, {q->loss, nullptr, nullptr}}, st);
}

int hiertcn_policy_loss(const hiertcn_rows_t* r, const hiertcn_policy_t* q, void* stream) {
  RowsP p{};
  int vec;
  if (!q) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  if (int rc = prepare(r, true, p, vec)) return rc;
  const hiertcn_rows_t& a = p.a;
  if (q->mean < 0 || q->mean > 1) return ops_fail(HIERTCN_ERR_INVALID, "mean %d: 0 over sequences, 1 over answers", q->mean);
  if (!(q->clip_low >= 0.f && q->clip_low <= 1.f) || !(q->clip_high >= 0.f && q->clip_high < 3e38f)) return ops_fail(HIERTCN_ERR_INVALID, "clip_low lies in [0, 1], clip_high is not negative");
  if (!(q->kl_coef >= 0.f && q->kl_coef < 3e38f)) return ops_fail(HIERTCN_ERR_INVALID, "kl_coef is not negative");
  if (!q->ref_logp && q->kl_coef != 0.f) return ops_fail(HIERTCN_ERR_INVALID, "kl_coef needs ref_logp");
  if (!q->old_logp || !q->advantage) return ops_fail(HIERTCN_ERR_INVALID, "null old_logp or advantage");
  if (q->adv_sn < 0 || q->adv_st < 0 || q->adv_sn > (1ll << 40) || q->adv_st > (1ll << 40)) return ops_fail(HIERTCN_ERR_INVALID, "a stride of advantage is negative");
  if ((uintptr_t)q->old_logp % 4 || (uintptr_t)q->ref_logp % 4 || (uintptr_t)q->advantage % 4) return ops_fail(HIERTCN_ERR_INVALID, "a pointer is not a multiple of 4");
  const OpsView ins[3] = {ops_flat(q->old_logp, p.R, 4), ops_flat(q->ref_logp, p.R, 4), OpsView{reinterpret_cast<const char*>(q->advantage), a.n, a.T, 1, q->adv_sn, q->adv_st, 4}};
  float* const outs[3] = {q->loss, q->kl, q->clipped};
  const char* const names[3] = {"loss", "kl", "clipped"};
  for (int i = 0; i < 3; i++) {
    if (int rc = check_out(p, outs[i], 1, names[i])) return rc;
    for (int j = 0; j < i; j++)
      if (outs[i] == outs[j]) return ops_fail(HIERTCN_ERR_INVALID, "%s overlaps %s", names[i], names[j]);
    for (const OpsView& v : ins)
      if (ops_overlap(ops_flat(outs[i], 1, 4), v)) return ops_fail(HIERTCN_ERR_INVALID, "%s overlaps an input", names[i]);
  }
  const OpsView lp = ops_flat(a.logp, p.R, 4);
  const OpsView d{static_cast<const char*>(a.dlogits), 1, p.R, a.V, 0, a.dld, ops_size(a.dtype)}, ws = ops_flat(a.workspace, (int64_t)a.workspace_bytes, 1);
  for (const OpsView& v : ins)
    if (ops_overlap(lp, v) || ops_overlap(d, v) || ops_overlap(ws, v)) return ops_fail(HIERTCN_ERR_INVALID, "logp, dlogits or the workspace overlaps an input");
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  ROWS_GO(k_part, p.R * p.parts + a.n, p);
  hipLaunchKernelGGL(k_policy, dim3((unsigned)((p.R + NT - 1) / NT)), dim3(NT), 0, st, p, *q);
  OPS_TRY(hipGetLastError());
  return finish(p, vec, Sums{p.term, p.R, 1.f, {q->loss, q->kl, q->clipped}}, st);
}

}  // extern "C"
