// Losses on the log-probabilities of answers, with their gradients to the logits (include/hiertcn_ops.h).
//
// Every loss here is a function of logp = z_y - m - ln s per row (m the row's largest logit, s = sum exp(z - m)), so its gradient to a row is
//   dz_j = c (  [j = y] - exp(z_j - m) / s ),   c = d loss / d logp,
// and a loss differs from another only in how c comes from the logp's.  Three launches:
//   k_part    one pass over the logits: (m, s) of every part of every row, running maximum and sum
//   k_pairs / k_policy / k_logp   a few lanes a row: joins its parts, forms logp; the loss and c, in 64 bits (they are few)
//   k_dlogits one pass over the logits: dz  (its first workgroup adds up the loss)
// Masked rows are not read: their gradient rows are written as zeros.  All sums run in a fixed order.
//
// Bound by memory: the answered rows are read twice (c needs a whole row, a pair's needs two sequences), all gradient rows written once.  64 x 30 x 300000 bf16,
// half of the rows answered: k_part 91 us for 0.58 GB (some of it in the last cache), k_policy 7, k_dlogits 280 for 1.73 GB (6.2 TB/s); 8 pairs x 30 x 300000
// fp32: 34, 9.8, 114.  At 16 pairs x 20 x 20778 bf16 and below it is three launches of 4 to 8 us.  (A single pass that keeps the rows in registers while their
// workgroups wait for one another is no faster: 461 us against 463 in two passes at the first of these, before the stores were taken past the caches.)
#include <math.h>

#include "ops.h"

namespace {

constexpr int NT = 256;                 // threads of a workgroup
constexpr int MAX_PARTS = 64;           // a wave joins a row's parts, one to a lane
constexpr int64_t MAX_V = 0x7fffffff - 4096;      // elements and vectors of a row are ints, and a thread's next ones are at most 4 NT behind the last

// how a row is split over workgroups
struct Cut {
  int parts;
  int64_t chunk;                        // vectors of a part
  int tpr;                              // threads of a part: NT, or a wave (four rows to a workgroup) where a row has few vectors
};
struct RowsP {
  hiertcn_rows_t a;
  int64_t R;
  Cut read, write;                      // k_part's and k_dlogits'
  float2* part;                         // [R][parts] (m, s)
  float2* stat;                         // [R] (m, 1 / s)
  float* coef;                          // [R] d (grad_scale * loss) / d logp
  double* term;                         // [3][groups] policy: weighted loss, kl, clipped of k_policy's workgroups
  int32_t* count;                       // [n] policy: answers of a sequence
  int64_t* total;                       // [counters][2] policy: answers, sequences with answers, of the workgroups that count
  int64_t groups, counters;
  int lanes;                            // lanes of k_pairs / k_policy / k_logp that join a row's parts: a power of two
};

__device__ __forceinline__ bool answered(const hiertcn_rows_t& a, int64_t r, int32_t& y) {
  y = a.ids[r];
  return y > 0 && y < a.V;
}

// (m, s) of two runs as one.  m = -inf: nothing in it (s is 0, or NaN and stays NaN).
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = ref_of(top);
  s = s * ops_exp_fp32(m - ref) + s2 * ops_exp_fp32(m2 - ref);
  m = top;
}
__device__ __forceinline__ void wave_join(float& m, float& s) {
#pragma unroll
  for (int d = 32; d; d >>= 1) join(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
}

// the part of a row as [head] vectors [tail]: head elements up to the first address that a vector may be loaded from.  (V <= MAX_V: ints.)
template <int DT, int VEC>
struct Span {
  int head, v0, v1;                     // v0 .. v1: this part's vectors; element of vector v: head + v * VEC
  int tail;                             // first element behind the vectors
  __device__ Span(const void* row, int V, int chunk, int part) {
    constexpr int ES = DT == HIERTCN_FP32 ? 4 : 2;
    head = VEC == 1 ? 0 : (int)((16 - ((uintptr_t)row & 15)) & 15) / ES;
    if (head > V) head = V;
    const int nvec = (V - head) / VEC;
    tail = head + nvec * VEC;
    v0 = part * chunk;
    v1 = nvec - v0 < chunk ? nvec : v0 + chunk;
  }
  // this thread's element in front of or behind the vectors, or -1 (there are at most VEC - 1 of each)
  __device__ int edge(int V, int part, int parts, int tid) const {
    if (part == 0 && tid < head) return tid;
    if (part == parts - 1 && tid >= 32 && tail + (tid - 32) < V) return tail + (tid - 32);
    return -1;
  }
};
template <int DT>
__device__ __forceinline__ const void* row_of(const void* p, int64_t off) {
  return DT == HIERTCN_FP32 ? (const void*)(static_cast<const float*>(p) + off) : (const void*)(static_cast<const uint16_t*>(p) + off);
}
template <int DT, int VEC>
__device__ __forceinline__ typename OpsRaw<DT, VEC>::type raw_at(const void* row, int e) {
  return *static_cast<const typename OpsRaw<DT, VEC>::type*>(row_of<DT>(row, e));
}
// which row and part this thread works on.  false: none
__device__ __forceinline__ bool place_of(const RowsP& p, const Cut& c, unsigned wg, int tpr, int64_t& r, int& part, int& tid) {
  tid = threadIdx.x & (tpr - 1);
  if (tpr == NT) {
    r = wg / (unsigned)c.parts;
    part = (int)(wg % (unsigned)c.parts);
  } else {                              // (one part)
    r = (int64_t)wg * (NT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    part = 0;
  }
  return r < p.R;
}

// U vectors' share of a running (m, s)
template <int DT, int VEC, int U>
__device__ __forceinline__ void fold(const typename OpsRaw<DT, VEC>::type (&x)[U], int live, float& m, float& s) {
  float z[U][VEC], top = m;
#pragma unroll
  for (int u = 0; u < U; u++) {
    ops_cvt<DT, VEC>(x[u], z[u]);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      if (u >= live) z[u][i] = -INFINITY;
      top = fmaxf(top, z[u][i]);
    }
  }
  const float ref = ref_of(top);
  s *= ops_exp_of<DT>(m - ref);
  m = top;
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < VEC; i++) s += ops_exp_of<DT>(z[u][i] - ref);
}

// answers per sequence, and this workgroup's share of their totals: a thread a sequence where sequences are short, else a wave
constexpr int COUNT_T = 64;
__device__ void count_answers(const RowsP& p, unsigned wg) {
  const hiertcn_rows_t& a = p.a;
  const int lane = threadIdx.x & 63;
  const bool thread = a.T <= COUNT_T;
  const int64_t q = thread ? (int64_t)wg * NT + threadIdx.x : (int64_t)wg * (NT / 64) + (threadIdx.x >> 6);
  int c = 0;
  if (q < a.n)
    for (int64_t t = thread ? 0 : lane; t < a.T; t += thread ? 1 : 64) {
      int32_t y;
      c += answered(a, q * a.T + t, y);
    }
  if (!thread)
#pragma unroll
    for (int d = 32; d; d >>= 1) c += __shfl_xor(c, d);
  const bool owner = q < a.n && (thread || lane == 0);
  if (owner) p.count[q] = c;
  int64_t all = owner ? c : 0;
  int some = owner && c > 0;
#pragma unroll
  for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d), some += __shfl_xor(some, d);
  __shared__ int64_t sums[NT / 64][2];
  if (lane == 0) sums[threadIdx.x >> 6][0] = all, sums[threadIdx.x >> 6][1] = some;
  __syncthreads();
  if (threadIdx.x < 2) p.total[2 * wg + threadIdx.x] = sums[0][threadIdx.x] + sums[1][threadIdx.x] + sums[2][threadIdx.x] + sums[3][threadIdx.x];
}

template <int DT, int VEC, int TPR>
__global__ __launch_bounds__(NT) void k_part(RowsP p) {
  constexpr int U = 4;
  const hiertcn_rows_t& a = p.a;
  if (blockIdx.x < p.counters) {
    count_answers(p, blockIdx.x);
    return;
  }
  int64_t r;
  int part, tid;
  int32_t y;
  if (!place_of(p, p.read, blockIdx.x - (unsigned)p.counters, TPR, r, part, tid) || !answered(a, r, y)) return;
  const void* row = row_of<DT>(a.logits, r * a.ld);
  const Span<DT, VEC> sp(row, (int)a.V, (int)p.read.chunk, part);
  float m = -INFINITY, s = 0.f;
  typename OpsRaw<DT, VEC>::type x[U];
  int v = sp.v0 + tid;
  const int full = sp.v1 > sp.v0 ? (sp.v1 - sp.v0) / (TPR * U) : 0;
  for (int k = 0; k < full; k++, v += TPR * U) {
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = raw_at<DT, VEC>(row, sp.head + (v + u * TPR) * VEC);
    fold<DT, VEC, U>(x, U, m, s);
  }
  if (v < sp.v1) {                                             // the rest: addresses behind it are clamped, their values not taken
    const int live = (sp.v1 - v + TPR - 1) / TPR;
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = raw_at<DT, VEC>(row, sp.head + (u < live ? v + u * TPR : v) * VEC);
    fold<DT, VEC, U>(x, live, m, s);
  }
  const int e = sp.edge((int)a.V, part, p.read.parts, tid);
  if (e >= 0) {
    float z[1];
    ops_ld<DT, 1>(row, e, z);
    join(m, s, z[0], z[0] == -INFINITY ? 0.f : 1.f + (z[0] - z[0]));
  }
  wave_join(m, s);
  if constexpr (TPR == NT) {
    __shared__ float ms[NT / 64], ss[NT / 64];
    if ((threadIdx.x & 63) == 0) ms[threadIdx.x >> 6] = m, ss[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 1; w < NT / 64; w++) join(m, s, ms[w], ss[w]);
  }
  if (tid == 0) p.part[r * p.read.parts + part] = make_float2(m, s);
}

__device__ __forceinline__ float logit(const hiertcn_rows_t& a, int64_t off) {
  return a.dtype == HIERTCN_FP32 ? static_cast<const float*>(a.logits)[off] : ops_h2f(static_cast<const uint16_t*>(a.logits)[off], a.dtype);
}

// p.lanes neighbours a row: logp from its parts, (m, 1 / s) kept for the gradient.  ROW_EMPTY: answered, but nothing but -inf
enum Row { ROW_MASKED, ROW_EMPTY, ROW_LIVE };
__device__ Row finish_row(const RowsP& p, int64_t r, double& logp) {
  int32_t y;
  logp = 0.0;
  if (!answered(p.a, r, y)) return ROW_MASKED;
  const int i = threadIdx.x & (p.lanes - 1);
  const float2 x = i < p.read.parts ? p.part[r * p.read.parts + i] : make_float2(-INFINITY, 0.f);
  const float z = logit(p.a, r * p.a.ld + y);
  float m = x.x, s = x.y;
  for (int d = p.lanes >> 1; d; d >>= 1) join(m, s, __shfl_xor(m, d), __shfl_xor(s, d));
  if (i == 0) p.stat[r] = make_float2(m, 1.f / s);
  if (m == -INFINITY && s == 0.f) return ROW_EMPTY;
  logp = ((double)z - ref_of(m)) - log((double)s);
  return ROW_LIVE;
}
// the row of this thread's lanes, of n rows beginning at the workgroup's first
__device__ __forceinline__ int64_t row_here(const RowsP& p) { return (int64_t)blockIdx.x * (NT / p.lanes) + threadIdx.x / p.lanes; }
__device__ __forceinline__ bool first_lane(const RowsP& p) { return (threadIdx.x & (p.lanes - 1)) == 0; }

__global__ __launch_bounds__(NT) void k_logp(RowsP p) {
  const int64_t r = row_here(p);
  if (r >= p.R) return;
  double lp;
  finish_row(p, r, lp);
  if (first_lane(p)) p.a.logp[r] = (float)lp;
}

// sums over a workgroup of W waves, for all its threads
template <int W, int N>
__device__ void block_sum(double (&x)[N]) {
  __shared__ double t[W][N];
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int d = 32; d; d >>= 1) x[k] += __shfl_xor(x[k], d);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++)
    if ((threadIdx.x & 63) == 0) t[threadIdx.x >> 6][k] = x[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++) {
    x[k] = t[0][k];
#pragma unroll
    for (int w = 1; w < W; w++) x[k] += t[w][k];
  }
}
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// loss and d loss / d D of a pair
__device__ __forceinline__ void pair_of(const hiertcn_preference_t& q, double D, double& loss, double& slope) {
  const double beta = q.beta, eps = q.smoothing;
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
}
// c of a sequence's rows, from the pair's slope
__device__ __forceinline__ float coef_of(const RowsP& p, const hiertcn_preference_t& q, double slope, int side, double count) {
  return (float)((side ? -slope : slope) / (double)(p.a.n / 2) * p.a.grad_scale / (q.average && count > 0 ? count : 1.0));
}

// a workgroup a pair: both sums, the loss, the rows' c.  (A thousand threads: the rows are a few hundred loads, one behind the other in a thread.)
constexpr int PAIR_NT = 1024;
__global__ __launch_bounds__(PAIR_NT) void k_pairs(RowsP p, hiertcn_preference_t q) {
  const hiertcn_rows_t& a = p.a;
  const int64_t P = a.n / 2;
  const int64_t first = threadIdx.x / p.lanes, step = PAIR_NT / p.lanes;
  const float ref[2] = {q.ref[blockIdx.x], q.ref[blockIdx.x + P]};
  double x[4] = {};                                            // sums of logp, numbers of answers
  uint64_t kept = 0;                                           // bit k: the k-th of this thread's rows has a distribution
  int k = 0;
  for (int64_t i = first; i < 2 * a.T; i += step, k++) {
    const int side = i >= a.T;
    const int64_t r = side ? (blockIdx.x + P) * a.T + (i - a.T) : blockIdx.x * a.T + i;
    double lp;
    const Row row = finish_row(p, r, lp);
    if (first_lane(p)) {
      a.logp[r] = (float)lp;
      if (k < 64) kept |= (uint64_t)(row == ROW_LIVE) << k;
      else p.coef[r] = row == ROW_LIVE ? 1.f : 0.f;
      const double one = row != ROW_MASKED ? 1.0 : 0.0;
      x[0] += side ? 0.0 : lp;
      x[1] += side ? lp : 0.0;
      x[2] += side ? 0.0 : one;
      x[3] += side ? one : 0.0;
    }
  }
  block_sum<PAIR_NT / 64>(x);
  __shared__ float c[2];
  if (threadIdx.x == 0) {                                      // one wave: 64-bit exponentials in all 16 cost 5 us
    double s[2];
    for (int side = 0; side < 2; side++) s[side] = q.average ? (x[2 + side] > 0 ? x[side] / x[2 + side] : 0.0) : x[side];
    const double D = (s[0] - ref[0]) - (s[1] - ref[1]);
    double loss, slope;
    pair_of(q, D, loss, slope);
    c[0] = coef_of(p, q, slope, 0, x[2]);
    c[1] = coef_of(p, q, slope, 1, x[3]);
    q.pair_loss[blockIdx.x] = (float)loss;
    q.margin[blockIdx.x] = (float)D;
    q.seq_logp[blockIdx.x] = (float)s[0];
    q.seq_logp[blockIdx.x + P] = (float)s[1];
  }
  __syncthreads();
  if (!first_lane(p)) return;
  k = 0;
  for (int64_t i = first; i < 2 * a.T; i += step, k++) {       // (this thread's own rows of the loop above)
    const int side = i >= a.T;
    const int64_t r = side ? (blockIdx.x + P) * a.T + (i - a.T) : blockIdx.x * a.T + i;
    const bool live = k < 64 ? kept >> k & 1 : p.coef[r] != 0.f;
    p.coef[r] = live ? c[side] : 0.f;
  }
}

// one answer of the policy loss: its weighted loss, kl and [clipped], and c without grad_scale
struct Answer { double loss, kl, cut, c; };
__device__ __forceinline__ Answer answer_of(const hiertcn_policy_t& q, int64_t T, int64_t r, double lp, double weight) {
  Answer o;
  const double A = q.advantage[r / T * q.adv_sn + r % T * q.adv_st];
  const double ratio = exp(lp - q.old_logp[r]);
  const double lo = 1.0 - q.clip_low, hi = 1.0 + q.clip_high;
  const double bounded = ratio < lo ? lo : ratio > hi ? hi : ratio;
  const double none = lp != lp ? lp : 0.0;      // 0, or the NaN of the row
  const double x = A == 0.0 ? none : ratio * A, y = A == 0.0 ? none : bounded * A;
  const bool clipped = x > y;
  o.loss = clipped ? -y : -x;
  o.cut = clipped ? weight : 0.0;
  o.c = clipped ? none : -x;
  o.kl = 0.0;
  if (q.ref_logp) {
    const double gap = q.ref_logp[r] - lp, e = expm1(gap);
    o.kl = e == INFINITY ? e : e - gap;
    if (q.kl_coef != 0.f) {             // (an infinite kl that is only looked at leaves the loss alone)
      o.loss += q.kl_coef * o.kl;
      o.c += q.kl_coef * -e;
    }
  }
  o.loss *= weight;
  o.kl *= weight;
  o.c *= weight;
  return o;
}

__global__ __launch_bounds__(NT) void k_policy(RowsP p, hiertcn_policy_t q) {
  const hiertcn_rows_t& a = p.a;
  double total[1] = {};                                        // sequences with answers, or answers
  for (int64_t i = threadIdx.x; i < p.counters; i += NT) total[0] += (double)p.total[2 * i + (q.mean == 0)];
  block_sum<NT / 64>(total);
  const int64_t r = row_here(p);
  double x[3] = {};
  if (r < p.R) {
    double lp;
    const bool live = finish_row(p, r, lp) == ROW_LIVE;
    if (first_lane(p)) {
      Answer o{0.0, 0.0, 0.0, 0.0};
      if (live) o = answer_of(q, a.T, r, lp, 1.0 / (q.mean == 0 ? total[0] * p.count[r / a.T] : total[0]));
      a.logp[r] = (float)lp;
      p.coef[r] = (float)(o.c * a.grad_scale);
      x[0] = o.loss, x[1] = o.kl, x[2] = o.cut;
    }
  }
  block_sum<NT / 64>(x);
  if (threadIdx.x < 3) p.term[threadIdx.x * p.groups + blockIdx.x] = threadIdx.x == 0 ? x[0] : threadIdx.x == 1 ? x[1] : x[2];
}

// out[k] = scale * sum of a row of n numbers, one workgroup
struct Sums { const float* f; const double* d; int64_t n; double scale; float* out[3]; };
__device__ void add_up(const Sums& q) {
  double x[3] = {};
  for (int64_t i = threadIdx.x; i < q.n; i += NT) {
    if (q.f) x[0] += q.f[i];
    else
#pragma unroll
      for (int k = 0; k < 3; k++) x[k] += q.d[k * q.n + i];
  }
  block_sum<NT / 64>(x);
#pragma unroll
  for (int k = 0; k < 3; k++)
    if (threadIdx.x == 0 && q.out[k]) q.out[k][0] = (float)(x[k] * q.scale);
}
__global__ __launch_bounds__(NT) void k_sums(Sums q) { add_up(q); }

template <int DT, int VEC>
__device__ __forceinline__ void gradient_of(const typename OpsRaw<DT, VEC>::type& x, void* out, int at, float ref, float g, float c, int y) {
  float z[VEC];
  ops_cvt<DT, VEC>(x, z);
#pragma unroll
  for (int i = 0; i < VEC; i++) z[i] = g * ops_exp_of<DT>(z[i] - ref);
  if (y >= at && y - at < VEC)
#pragma unroll
    for (int i = 0; i < VEC; i++) z[i] += i == y - at ? c : 0.f;
  ops_st<DT, VEC, true>(out, at, z);
}

template <int DT, int VEC, int TPR>
__global__ __launch_bounds__(NT) void k_dlogits(RowsP p, Sums q) {
  constexpr int U = 4;
  const hiertcn_rows_t& a = p.a;
  if (blockIdx.x == 0) {
    add_up(q);
    return;
  }
  int64_t r;
  int part, tid;
  // backwards: k_part's last rows may still be in the last level of cache.  Its lines are not kept for the stores' sake (64 x 30 x 300000 bf16, both
  // passes: 546 us; stores past the caches 520, backwards 525, both 501)
  if (!place_of(p, p.write, gridDim.x - 1 - blockIdx.x, TPR, r, part, tid)) return;
  const float c = p.coef[r];
  const float2 st = p.stat[r];                                 // (not written for a masked row, and not used)
  const int y = a.ids[r];
  const void* row = row_of<DT>(a.logits, r * a.ld);
  void* out = const_cast<void*>(row_of<DT>(a.dlogits, r * a.dld));
  const Span<DT, VEC> sp(out, (int)a.V, (int)p.write.chunk, part);
  const int e = sp.edge((int)a.V, part, p.write.parts, tid);
  int v = sp.v0 + tid;
  if (c == 0.f) {
    const float zero[VEC] = {};
    for (; v < sp.v1; v += TPR) ops_st<DT, VEC, true>(out, sp.head + v * VEC, zero);
    const float z1[1] = {0.f};
    if (e >= 0) ops_st<DT, 1>(out, e, z1);
    return;
  }
  const float ref = ref_of(st.x), g = -c * st.y;
  typename OpsRaw<DT, VEC>::type x[U];
  const int full = sp.v1 > sp.v0 ? (sp.v1 - sp.v0) / (TPR * U) : 0;
  for (int k = 0; k < full; k++, v += TPR * U) {
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = raw_at<DT, VEC>(row, sp.head + (v + u * TPR) * VEC);
#pragma unroll
    for (int u = 0; u < U; u++) gradient_of<DT, VEC>(x[u], out, sp.head + (v + u * TPR) * VEC, ref, g, c, y);
  }
  if (v < sp.v1) {
    const int live = (sp.v1 - v + TPR - 1) / TPR;
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = raw_at<DT, VEC>(row, sp.head + (u < live ? v + u * TPR : v) * VEC);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (u < live) gradient_of<DT, VEC>(x[u], out, sp.head + (v + u * TPR) * VEC, ref, g, c, y);
  }
  if (e >= 0) {
    float z[1];
    ops_ld<DT, 1>(row, e, z);
    z[0] = g * ops_exp_of<DT>(z[0] - ref);
    if (e == y) z[0] += c;
    ops_st<DT, 1>(out, e, z);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------------------
size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
// parts of `elems` elements, or of as many more as MAX_PARTS asks for.  A wave for a row that one round of its loads covers, or four rounds where there are rows
// enough to fill the machine with waves; else a workgroup (12800 rows, both passes, us, wave / workgroup: 1000 bf16 25 / 42, 2000 32 / 51, 4000 49 / 65, 8000 84 / 88)
Cut cut_of(int64_t R, int64_t V, int vec, int64_t elems) {
  if ((V + elems - 1) / elems > MAX_PARTS) elems = (V + MAX_PARTS - 1) / MAX_PARTS;
  Cut c;
  c.chunk = (elems + vec - 1) / vec;
  const int64_t nvec = V / vec;
  c.parts = (int)(nvec <= c.chunk ? 1 : (nvec + c.chunk - 1) / c.chunk);
  c.tpr = c.parts == 1 && (nvec <= 256 || (nvec <= 1024 && R >= 4096)) ? 64 : NT;
  return c;
}
// (64 x 30 x 300000 bf16 and 16 x 30 x 300000 fp32: parts of 4096 to 16384 elements are within 2 % for the second pass, 32768 2 to 4 % slower)
constexpr int64_t PART = 8192;
// k_part's parts grow while 8192 of them are left (fewer prologues and joins: 148 us against 155 at 64 x 30 x 300000 bf16)
Cut read_of(int64_t R, int64_t V, int vec) {
  int64_t elems = PART;
  while (elems < 4 * PART && R * ((V + 2 * elems - 1) / (2 * elems)) >= 8192) elems *= 2;
  return cut_of(R, V, vec, elems);
}
int64_t workgroups(const Cut& c, int64_t R) { return c.tpr == NT ? R * c.parts : (R + NT / 64 - 1) / (NT / 64); }
int64_t counters_of(int64_t n, int64_t T) { return T <= COUNT_T ? (n + NT - 1) / NT : (n + NT / 64 - 1) / (NT / 64); }
size_t workspace_of(int64_t n, int64_t T, int64_t V, RowsP* p) {
  const size_t R = (size_t)(n * T);
  int most = 1;
  for (int vec : {1, 4, 8}) most = most > read_of(n * T, V, vec).parts ? most : read_of(n * T, V, vec).parts;
  int lanes = 1;
  while (lanes < most) lanes *= 2;
  const size_t groups = (R + NT / lanes - 1) / (NT / lanes);
  const size_t sizes[6] = {align_up(R * most * 8), align_up(R * 8), align_up(R * 4), align_up(groups * 24), align_up((size_t)n * 4), align_up((size_t)counters_of(n, T) * 16)};
  if (p) {
    p->lanes = lanes;
    p->groups = (int64_t)groups;
  }
  if (p && p->a.workspace) {
    char* w = static_cast<char*>(p->a.workspace);
    p->part = reinterpret_cast<float2*>(w);
    p->stat = reinterpret_cast<float2*>(w += sizes[0]);
    p->coef = reinterpret_cast<float*>(w += sizes[1]);
    p->term = reinterpret_cast<double*>(w += sizes[2]);
    p->count = reinterpret_cast<int32_t*>(w += sizes[3]);
    p->total = reinterpret_cast<int64_t*>(w += sizes[4]);
  }
  return sizes[0] + sizes[1] + sizes[2] + sizes[3] + sizes[4] + sizes[5];
}

// the checks that all entries share; sets up p
int prepare(const hiertcn_rows_t* in, bool grad, RowsP& p, int& vec) {
  if (!in) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  p.a = *in;
  hiertcn_rows_t& a = p.a;
  if (!grad) a.dlogits = nullptr;
  if (a.n < 1 || a.T < 1 || a.V < 1) return ops_fail(HIERTCN_ERR_INVALID, "n, T and V are at least 1 (%lld, %lld, %lld)", (long long)a.n, (long long)a.T, (long long)a.V);
  if (a.n > (1ll << 31) || a.T > (1ll << 31) || a.n * a.T > (1ll << 31) || a.V > MAX_V) return ops_fail(HIERTCN_ERR_INVALID, "n * T is at most 2^31, V at most 2^31 - 4097");
  if (!ops_dtype_ok(a.dtype)) return ops_fail(HIERTCN_ERR_INVALID, "dtype %d: 0 fp32, 1 bf16, 2 fp16", a.dtype);
  if (!a.logits || !a.ids || !a.logp) return ops_fail(HIERTCN_ERR_INVALID, "null logits, ids or logp");
  p.R = a.n * a.T;
  if (p.R == 1) a.ld = a.V, a.dld = a.dlogits ? a.V : 0;
  if (a.ld < a.V || a.ld > (1ll << 40) || (a.dlogits && (a.dld < a.V || a.dld > (1ll << 40)))) return ops_fail(HIERTCN_ERR_INVALID, "a row stride is smaller than V");
  const int es = ops_size(a.dtype);
  // 16 bytes at a time wherever the two passes' rows are 16-byte aligned alike; else one element
  vec = 16 / es;
  if (a.dlogits && (((uintptr_t)a.logits - (uintptr_t)a.dlogits) % 16 || (a.ld - a.dld) % vec)) vec = 1;
  p.read = read_of(p.R, a.V, vec);
  p.write = cut_of(p.R, a.V, vec, PART);
  p.counters = 0;
  workspace_of(a.n, a.T, a.V, &p);      // (addresses into a workspace that is checked below)
  const int64_t most = ops_most_groups(NT);
  if (workgroups(p.read, p.R) + counters_of(a.n, a.T) > most || workgroups(p.write, p.R) + 1 > most || p.groups > most)
    return ops_fail(HIERTCN_ERR_INVALID, "%lld rows of %lld are too many for one launch: at most 2^24 - 1 workgroups of a part of a row, or of four short rows", (long long)p.R, (long long)a.V);
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
  return HIERTCN_OK;
}

#define ROWS_VEC(kernel, dt, wide, tpr, g, ...)                                                                                                \
  do {                                                                                                                                         \
    if (vec == 1 && tpr == NT) hipLaunchKernelGGL((kernel<dt, 1, NT>), g, dim3(NT), 0, st, __VA_ARGS__);                                        \
    else if (vec == 1) hipLaunchKernelGGL((kernel<dt, 1, 64>), g, dim3(NT), 0, st, __VA_ARGS__);                                                \
    else if (tpr == NT) hipLaunchKernelGGL((kernel<dt, wide, NT>), g, dim3(NT), 0, st, __VA_ARGS__);                                            \
    else hipLaunchKernelGGL((kernel<dt, wide, 64>), g, dim3(NT), 0, st, __VA_ARGS__);                                                           \
  } while (0)
#define ROWS_GO(kernel, cut, extra, ...)                                                                                                       \
  do {                                                                                                                                         \
    const dim3 g_((unsigned)(workgroups(cut, p.R) + (extra)));                                                                                 \
    if (p.a.dtype == HIERTCN_FP32) ROWS_VEC(kernel, HIERTCN_FP32, 4, cut.tpr, g_, __VA_ARGS__);                                                 \
    else if (p.a.dtype == HIERTCN_BF16) ROWS_VEC(kernel, HIERTCN_BF16, 8, cut.tpr, g_, __VA_ARGS__);                                            \
    else ROWS_VEC(kernel, HIERTCN_FP16, 8, cut.tpr, g_, __VA_ARGS__);                                                                           \
    OPS_TRY(hipGetLastError());                                                                                                                \
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
    ROWS_GO(k_dlogits, p.write, 1, p, s);
  } else {
    hipLaunchKernelGGL(k_sums, dim3(1), dim3(NT), 0, st, s);
    OPS_TRY(hipGetLastError());
  }
  return HIERTCN_OK;
}

}  // namespace

extern "C" {

size_t hiertcn_rows_workspace_bytes(int64_t n, int64_t T, int64_t V) {
  return n < 1 || T < 1 || V < 1 || n > (1ll << 31) || T > (1ll << 31) || n * T > (1ll << 31) || V > MAX_V ? 0 : workspace_of(n, T, V, nullptr);
}

int hiertcn_sequence_logp(const hiertcn_rows_t* r, void* stream) {
  RowsP p{};
  int vec;
  if (int rc = prepare(r, false, p, vec)) return rc;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  ROWS_GO(k_part, p.read, 0, p);
  hipLaunchKernelGGL(k_logp, dim3((unsigned)p.groups), dim3(NT), 0, st, p);
  OPS_TRY(hipGetLastError());
  return HIERTCN_OK;
}

int hiertcn_preference_loss(const hiertcn_rows_t* r, const hiertcn_preference_t* q, void* stream) {
  RowsP p{};
  int vec;
  if (!q) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  if (int rc = prepare(r, true, p, vec)) return rc;
  const int64_t n = p.a.n, P = n / 2;
  if (P > ops_most_groups(PAIR_NT)) return ops_fail(HIERTCN_ERR_INVALID, "%lld pairs: at most 2^22 - 1", (long long)P);
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
  ROWS_GO(k_part, p.read, 0, p);
  hipLaunchKernelGGL(k_pairs, dim3((unsigned)P), dim3(PAIR_NT), 0, st, p, *q);
  OPS_TRY(hipGetLastError());
  return finish(p, vec, Sums{q->pair_loss, nullptr, P, 1.0 / (double)P, {q->loss, nullptr, nullptr}}, st);
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
  p.counters = counters_of(a.n, a.T);
  ROWS_GO(k_part, p.read, p.counters, p);
  hipLaunchKernelGGL(k_policy, dim3((unsigned)p.groups), dim3(NT), 0, st, p, *q);
  OPS_TRY(hipGetLastError());
  return finish(p, vec, Sums{nullptr, p.term, p.groups, 1.0, {q->loss, q->kl, q->clipped}}, st);
}

}  // extern "C"
