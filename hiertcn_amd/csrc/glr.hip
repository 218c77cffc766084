// Gated linear recurrence (include/hiertcn_ops.h): h_t = u_t [keep_t] h_{t-1} + (1 - u_t) c_t with u = sigmoid(gate) and c = cand or tanh(cand) --
// the update of customed_gru_cell.py:309-337 with gates that do not read the state, hence a scan.
//
// The map of a run of steps is h -> A h + S (A the product of the a_t = u_t keep_t, S the run's own state from zero), and maps compose:
// (A2, S2) after (A1, S1) is (A2 A1, A2 S1 + S2).  Time is cut into SEGMENTS of 8 steps; a thread owns a segment of VEC neighbouring channels and
// keeps its a_t and (1 - u_t) c_t in registers, so that gate and cand are read once: it forms (A, S), learns the state before its segment from the maps
// of the segments before it (lanes of a wave by shuffles, waves of a workgroup through LDS, earlier tiles as a carry in registers, earlier
// workgroups through `agg`), and replays the segment from there.
//
// The backward pass is the same recurrence the other way round, lambda_t = dout_t + a_{t+1} lambda_{t+1}: with r_t = a_t lambda_t a run maps r -> A r + Q
// with the same A.  States are not read back from the rounded output: the forward pass leaves the fp32 state before every segment in `record`, 1/8 of
// a [B][T][D] fp32 array, and a thread replays its segment from there.
//
// A reset has to cut a state that is NaN or infinite (0 * NaN = NaN), and nothing else may: A is exactly 0 only where a reset lies in the run (the
// product of the gates alone is kept from underflowing to 0), and a map with A = 0 ignores what it is applied to.
#include "ops.h"

namespace {

constexpr int SEG = 8;           // steps of a segment = distance of the records
constexpr int CB = 64;           // channels of a workgroup
constexpr float TINY = 1.401298464e-45f;

struct GlrP {
  hiertcn_glr_t a;
  int64_t nseg;                  // ceil(T / SEG)
  int ncb;                       // channel blocks
  int nchunk, chunk_tiles;       // the time axis over several workgroups
  float2* agg;                   // [nchunk][B][D]: the chunks' maps
  float* state0;                 // [B][D] copy of state_in (state_out may be state_in) when nchunk > 1
};

struct Map { float A, S; };
__device__ __forceinline__ float map_a(float A1, float A2) { return A1 == 0.f || A2 == 0.f ? 0.f : fmaxf(A1 * A2, TINY); }
__device__ __forceinline__ float map_s(float A2, float S1, float S2) { return A2 == 0.f ? S2 : fmaf(A2, S1, S2); }

// u = sigmoid(g) and w = 1 - u = sigmoid(-g), each to a few ulp (1 - u formed from u would lose the small ones)
__device__ __forceinline__ void gate_of(float g, float& u, float& w) {
  const float e = ops_exp(-fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.f + e);
  u = g >= 0.f ? r : e * r;
  w = g >= 0.f ? e * r : r;
  if (g != g) u = w = g;
}
// tanh to a few ulp: the odd series where (1 - e^-2x) / (1 + e^-2x) would cancel
__device__ __forceinline__ float tanh_of(float x) {
  const float a = fabsf(x), x2 = x * x;
  const float e = ops_exp(-2.f * a);
  const float big = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
  float s = fmaf(x2, -8.863235530e-3f, 2.186948854e-2f);     // x - x^3/3 + 2x^5/15 - 17x^7/315 + 62x^9/2835 - 1382x^11/155925
  s = fmaf(x2, s, -5.396825397e-2f);
  s = fmaf(x2, s, 1.333333333e-1f);
  s = fmaf(x2, s, -3.333333333e-1f);
  return a < 0.3f ? fmaf(x * x2, s, x) : big;
}

// what a thread knows of its place
template <int VEC>
struct Place {
  static constexpr int CL = CB / VEC, TS = 64 / CL;
  int64_t b, ch;                 // lane (sequence) and first channel
  bool chan;                     // the channels exist
  int len;                       // steps of the sequence that count
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ int64_t length_of(const hiertcn_glr_t& a, int64_t b) { return a.lengths ? clamp64(a.lengths[b], 0, a.T) : a.T; }

// bits of the steps t0 .. t0 + n - 1 whose state is kept (steps behind the end keep it)
__device__ __forceinline__ uint32_t keep_bits(const hiertcn_glr_t& a, int64_t b, int64_t t0, int n) {
  uint32_t k = 0xffffffffu;
  if (a.mask) {
    const float* m = a.mask + b * a.mask_sb + t0 * a.mask_st;
    for (int j = 0; j < n; j++)
      if (m[j * a.mask_st] == 0.f) k &= ~(1u << j);
  }
  return k;
}

// Loads the gates (and candidates) of a segment with n >= 1 live steps; a dead step repeats the last live one's address.
template <int DT, int VEC>
__device__ __forceinline__ void load_rows(const void* p, int64_t base, int64_t st, int n, float (&o)[SEG][VEC]) {
  if (__all(n == SEG)) {
#pragma unroll
    for (int j = 0; j < SEG; j++) ops_ld<DT, VEC>(p, base + j * st, o[j]);
  } else {
#pragma unroll
    for (int j = 0; j < SEG; j++) ops_ld<DT, VEC>(p, base + (j < n ? j : n - 1) * st, o[j]);
  }
}

// a_t and b_t = w_t c_t of a segment (identity steps behind n)
template <int DT, int VEC, bool TANH>
__device__ __forceinline__ void load_forward(const hiertcn_glr_t& a, int64_t b, int64_t t0, int64_t ch, int n, float (&u)[SEG][VEC], float (&s)[SEG][VEC]) {
  if (n > 0) {
    load_rows<DT, VEC>(a.gate, b * a.gate_sb + t0 * a.gate_st + ch, a.gate_st, n, u);
    load_rows<DT, VEC>(a.cand, b * a.cand_sb + t0 * a.cand_st + ch, a.cand_st, n, s);
  }
#pragma unroll
  for (int j = 0; j < SEG; j++)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      if (j < n) {
        float w;
        gate_of(u[j][i], u[j][i], w);
        s[j][i] = w * (TANH ? tanh_of(s[j][i]) : s[j][i]);
      } else {
        u[j][i] = 1.f;
        s[j][i] = 0.f;
      }
    }
}
template <int VEC>
__device__ __forceinline__ void segment_map(const float (&u)[SEG][VEC], const float (&s)[SEG][VEC], uint32_t keep, float (&A)[VEC], float (&S)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i++) A[i] = 1.f, S[i] = 0.f;
#pragma unroll
  for (int j = 0; j < SEG; j++)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      S[i] = keep >> j & 1 ? fmaf(u[j][i], S[i], s[j][i]) : s[j][i];
      A[i] *= u[j][i];
    }
#pragma unroll
  for (int i = 0; i < VEC; i++) A[i] = keep == 0xffffffffu ? (A[i] == A[i] ? fmaxf(A[i], TINY) : A[i]) : 0.f;
}
// replays a segment from the state h, writing nrow output rows
template <int DT, int VEC>
__device__ __forceinline__ void replay(const hiertcn_glr_t& a, int64_t b, int64_t t0, int64_t ch, bool chan, int n, int nrow, uint32_t keep, const float (&u)[SEG][VEC],
                                       const float (&s)[SEG][VEC], float (&h)[VEC]) {
  const int64_t base = b * a.out_sb + t0 * a.out_st + ch;
#pragma unroll
  for (int j = 0; j < SEG; j++) {
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      h[i] = keep >> j & 1 ? fmaf(u[j][i], h[i], s[j][i]) : s[j][i];
      o[i] = j < n ? h[i] : 0.f;
    }
    if (j < nrow && chan) ops_st<DT, VEC>(a.out, base + j * a.out_st, o);
  }
}
template <int VEC>
__device__ __forceinline__ void get_state(const float* p, int64_t b, int64_t D, int64_t ch, float (&h)[VEC]) {
  if (p) ops_ld<HIERTCN_FP32, VEC>(p, b * D + ch, h);
  else
#pragma unroll
    for (int i = 0; i < VEC; i++) h[i] = 0.f;
}

// ---- forward, one thread a sequence's channels, segment after segment: many lanes, or few steps --------------------------------------------------
template <int DT, int VEC, bool TANH>
__global__ __launch_bounds__(64) void k_glr_seq(GlrP p) {
  const hiertcn_glr_t& a = p.a;
  const int64_t groups = a.D / VEC, id = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (id >= a.B * groups) return;
  const int64_t b = id / groups, ch = id % groups * VEC;
  const int64_t len = length_of(a, b);
  float h[VEC], u[SEG][VEC], s[SEG][VEC];
  get_state<VEC>(a.state_in, b, a.D, ch, h);
  for (int64_t g = 0; g < p.nseg; g++) {
    const int64_t t0 = g * SEG;
    const int n = (int)clamp64(len - t0, 0, SEG), nrow = (int)clamp64(a.T - t0, 0, SEG);
    if (a.record) ops_st<HIERTCN_FP32, VEC>(a.record, (b * p.nseg + g) * a.D + ch, h);
    load_forward<DT, VEC, TANH>(a, b, t0, ch, n, u, s);
    const uint32_t keep = keep_bits(a, b, t0, n);
    replay<DT, VEC>(a, b, t0, ch, true, n, nrow, keep, u, s, h);
  }
  if (a.state_out) ops_st<HIERTCN_FP32, VEC>(a.state_out, b * a.D + ch, h);
}

// ---- the maps of a workgroup's segments ---------------------------------------------------------------------------------------------------------
// In: this thread's map.  Out: the state before (REV: behind) its segment, given `carry` before the tile, and `carry` behind it.  One barrier; `lds`
// alternates between two buffers, so that the next tile's writes need no second one.
template <int VEC, bool REV>
__device__ __forceinline__ void tile_scan(float2* lds, int nw, int w, int ts, int cl, const float (&A)[VEC], const float (&S)[VEC], float (&carry)[VEC], float (&h)[VEC]) {
  constexpr int CL = CB / VEC, TS = 64 / CL;
  const int order = REV ? TS - 1 - ts : ts;
  float IA[VEC], IS[VEC];          // the maps of the wave's segments up to and with this one
#pragma unroll
  for (int i = 0; i < VEC; i++) IA[i] = A[i], IS[i] = S[i];
#pragma unroll
  for (int d = 1; d < TS; d <<= 1)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const float pa = REV ? __shfl_down(IA[i], d * CL) : __shfl_up(IA[i], d * CL), ps = REV ? __shfl_down(IS[i], d * CL) : __shfl_up(IS[i], d * CL);
      if (order >= d) {
        IS[i] = map_s(IA[i], ps, IS[i]);
        IA[i] = map_a(pa, IA[i]);
      }
    }
  if (order == TS - 1)
#pragma unroll
    for (int i = 0; i < VEC; i++) lds[w * CB + cl * VEC + i] = make_float2(IA[i], IS[i]);
  float XA[VEC], XS[VEC];          // ... before this one
#pragma unroll
  for (int i = 0; i < VEC; i++) {
    const float pa = REV ? __shfl_down(IA[i], CL) : __shfl_up(IA[i], CL), ps = REV ? __shfl_down(IS[i], CL) : __shfl_up(IS[i], CL);
    XA[i] = order ? pa : 1.f;
    XS[i] = order ? ps : 0.f;
  }
  __syncthreads();
  for (int q = 0; q < nw; q++) {
    const int ww = REV ? nw - 1 - q : q;
    if (ww == w)
#pragma unroll
      for (int i = 0; i < VEC; i++) h[i] = map_s(XA[i], carry[i], XS[i]);
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const float2 m = lds[ww * CB + cl * VEC + i];
      carry[i] = map_s(m.x, carry[i], m.y);
    }
  }
}

// ---- forward, a workgroup 64 channels of a sequence and a tile of nw * TS segments at a time --------------------------------------------------------
// AGG: only the map of the chunk is wanted (first pass of a time axis that is cut over workgroups).
template <int DT, int VEC, bool TANH, bool AGG>
__global__ __launch_bounds__(1024) void k_glr_tile(GlrP p) {
  constexpr int CL = CB / VEC, TS = 64 / CL;
  __shared__ float2 lds[2][16 * CB];
  const hiertcn_glr_t& a = p.a;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, ts = lane / CL, cl = lane % CL;
  const int64_t blk = blockIdx.x, cb = blk % p.ncb, b = blk / p.ncb % a.B, chunk = blk / p.ncb / a.B;
  const bool chan = cb * CB + cl * VEC < a.D;
  const int64_t ch = chan ? cb * CB + cl * VEC : 0;
  const int64_t len = length_of(a, b);
  const int tile_seg = nw * TS;
  const int64_t seg0 = chunk * p.chunk_tiles * tile_seg;
  const int64_t seg1 = p.nchunk > 1 && chunk + 1 < p.nchunk ? seg0 + (int64_t)p.chunk_tiles * tile_seg : p.nseg;
  float carry[VEC], carryA[VEC], h[VEC], u[SEG][VEC], s[SEG][VEC], A[VEC], S[VEC];
  if (AGG) {
#pragma unroll
    for (int i = 0; i < VEC; i++) carry[i] = 0.f, carryA[i] = 1.f;
    if (chunk == 0 && w == 0 && ts == 0 && chan) {
      get_state<VEC>(a.state_in, b, a.D, ch, h);
      ops_st<HIERTCN_FP32, VEC>(p.state0, b * a.D + ch, h);
    }
  } else if (p.nchunk > 1) {
    get_state<VEC>(p.state0, b, a.D, ch, carry);
    for (int64_t q = 0; q < chunk; q++)
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const float2 m = p.agg[(q * a.B + b) * a.D + ch + i];
        carry[i] = map_s(m.x, carry[i], m.y);
      }
  } else {
    get_state<VEC>(a.state_in, b, a.D, ch, carry);
  }
  int turn = 0;
  for (int64_t g0 = seg0; g0 < seg1; g0 += tile_seg, turn ^= 1) {
    const int64_t g = g0 + w * TS + ts, t0 = g * SEG;
    const int n = (int)clamp64(len - t0, 0, SEG), nrow = g < seg1 ? (int)clamp64(a.T - t0, 0, SEG) : 0;
    if (AGG && g0 * SEG >= len) break;       // (len is the workgroup's)
    load_forward<DT, VEC, TANH>(a, b, t0, ch, n, u, s);
    const uint32_t keep = keep_bits(a, b, t0, n);
    segment_map<VEC>(u, s, keep, A, S);
    if (AGG) {
#pragma unroll
      for (int i = 0; i < VEC; i++) h[i] = A[i];
      float before[VEC];
      tile_scan<VEC, false>(lds[turn], nw, w, ts, cl, A, S, carry, before);
      for (int q = 0; q < nw; q++)
#pragma unroll
        for (int i = 0; i < VEC; i++) carryA[i] = map_a(carryA[i], lds[turn][q * CB + cl * VEC + i].x);
      continue;
    }
    tile_scan<VEC, false>(lds[turn], nw, w, ts, cl, A, S, carry, h);
    if (a.record && nrow > 0 && chan) ops_st<HIERTCN_FP32, VEC>(a.record, (b * p.nseg + g) * a.D + ch, h);
    replay<DT, VEC>(a, b, t0, ch, chan, n, nrow, keep, u, s, h);
  }
  if (w != 0 || ts != 0 || !chan) return;
  if (AGG) {
#pragma unroll
    for (int i = 0; i < VEC; i++) p.agg[(chunk * a.B + b) * a.D + ch + i] = make_float2(carryA[i], carry[i]);
  } else if (a.state_out && chunk == p.nchunk - 1) {
    ops_st<HIERTCN_FP32, VEC>(a.state_out, b * a.D + ch, carry);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------------------------
// Per element of a segment: u, fg = (h_prev - c) u (1 - u) and fx = (1 - u) act'(c), so that dgate = lambda fg and dcand = lambda fx; d = dout.
// h: the state before the segment (the record).
template <int DT, int VEC, bool TANH>
__device__ __forceinline__ void load_backward(const hiertcn_glr_t& a, int64_t b, int64_t t0, int64_t ch, int n, uint32_t keep, float (&h)[VEC], float (&u)[SEG][VEC],
                                              float (&fg)[SEG][VEC], float (&fx)[SEG][VEC], float (&d)[SEG][VEC]) {
  if (n > 0) {
    load_rows<DT, VEC>(a.gate, b * a.gate_sb + t0 * a.gate_st + ch, a.gate_st, n, u);
    load_rows<DT, VEC>(a.cand, b * a.cand_sb + t0 * a.cand_st + ch, a.cand_st, n, fx);
    load_rows<DT, VEC>(a.dout, b * a.dout_sb + t0 * a.dout_st + ch, a.dout_st, n, d);
  }
#pragma unroll
  for (int j = 0; j < SEG; j++)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      if (j < n) {
        float w;
        gate_of(u[j][i], u[j][i], w);
        const float c = TANH ? tanh_of(fx[j][i]) : fx[j][i];
        const float hp = keep >> j & 1 ? h[i] : 0.f;
        h[i] = fmaf(u[j][i], hp, w * c);
        fg[j][i] = (hp - c) * (u[j][i] * w);
        fx[j][i] = TANH ? w * fmaf(-c, c, 1.f) : w;
      } else {
        u[j][i] = 1.f;
        fg[j][i] = fx[j][i] = d[j][i] = 0.f;
      }
    }
}
// r -> A r + Q of a segment, last step first
template <int VEC>
__device__ __forceinline__ void segment_map_rev(const float (&u)[SEG][VEC], const float (&d)[SEG][VEC], uint32_t keep, float (&A)[VEC], float (&Q)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i++) A[i] = 1.f, Q[i] = 0.f;
#pragma unroll
  for (int j = SEG - 1; j >= 0; j--)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      Q[i] = keep >> j & 1 ? u[j][i] * (d[j][i] + Q[i]) : 0.f;
      A[i] *= u[j][i];
    }
#pragma unroll
  for (int i = 0; i < VEC; i++) A[i] = keep == 0xffffffffu ? (A[i] == A[i] ? fmaxf(A[i], TINY) : A[i]) : 0.f;
}
// gradients of a segment, given r behind it; r before it afterwards
template <int DT, int VEC>
__device__ __forceinline__ void replay_rev(const hiertcn_glr_t& a, int64_t b, int64_t t0, int64_t ch, bool chan, int n, int nrow, uint32_t keep, const float (&u)[SEG][VEC],
                                           const float (&fg)[SEG][VEC], const float (&fx)[SEG][VEC], const float (&d)[SEG][VEC], float (&r)[VEC]) {
  const int64_t bg = b * a.dgate_sb + t0 * a.dgate_st + ch, bc = b * a.dcand_sb + t0 * a.dcand_st + ch;
#pragma unroll
  for (int j = SEG - 1; j >= 0; j--) {
    float og[VEC], oc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const float lam = d[j][i] + r[i];
      og[i] = j < n ? lam * fg[j][i] : 0.f;
      oc[i] = j < n ? lam * fx[j][i] : 0.f;
      r[i] = keep >> j & 1 ? u[j][i] * lam : 0.f;      // (a step behind the end has u = 1, d = 0: r passes)
    }
    if (j < nrow && chan) {
      ops_st<DT, VEC>(a.dgate, bg + j * a.dgate_st, og);
      ops_st<DT, VEC>(a.dcand, bc + j * a.dcand_st, oc);
    }
  }
}

template <int DT, int VEC, bool TANH>
__global__ __launch_bounds__(64) void k_glr_seq_bwd(GlrP p) {
  const hiertcn_glr_t& a = p.a;
  const int64_t groups = a.D / VEC, id = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (id >= a.B * groups) return;
  const int64_t b = id / groups, ch = id % groups * VEC;
  const int64_t len = length_of(a, b);
  float r[VEC], h[VEC], u[SEG][VEC], fg[SEG][VEC], fx[SEG][VEC], d[SEG][VEC];
  get_state<VEC>(a.dstate_out, b, a.D, ch, r);
  for (int64_t g = p.nseg - 1; g >= 0; g--) {
    const int64_t t0 = g * SEG;
    const int n = (int)clamp64(len - t0, 0, SEG), nrow = (int)clamp64(a.T - t0, 0, SEG);
    get_state<VEC>(a.record + g * a.D, b, p.nseg * a.D, ch, h);
    const uint32_t keep = keep_bits(a, b, t0, n);
    load_backward<DT, VEC, TANH>(a, b, t0, ch, n, keep, h, u, fg, fx, d);
    replay_rev<DT, VEC>(a, b, t0, ch, true, n, nrow, keep, u, fg, fx, d, r);
  }
  if (a.dstate_in) ops_st<HIERTCN_FP32, VEC>(a.dstate_in, b * a.D + ch, r);
}

template <int DT, int VEC, bool TANH>
__global__ __launch_bounds__(1024) void k_glr_tile_bwd(GlrP p) {
  constexpr int CL = CB / VEC, TS = 64 / CL;
  __shared__ float2 lds[2][16 * CB];
  const hiertcn_glr_t& a = p.a;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, ts = lane / CL, cl = lane % CL;
  const int64_t blk = blockIdx.x, cb = blk % p.ncb, b = blk / p.ncb % a.B, chunk = blk / p.ncb / a.B;
  const bool chan = cb * CB + cl * VEC < a.D;
  const int64_t ch = chan ? cb * CB + cl * VEC : 0;
  const int64_t len = length_of(a, b);
  const int tile_seg = nw * TS;
  const int64_t seg0 = chunk * p.chunk_tiles * tile_seg;
  const int64_t seg1 = chunk + 1 < p.nchunk ? seg0 + (int64_t)p.chunk_tiles * tile_seg : p.nseg;
  const int64_t tiles = (seg1 - seg0 + tile_seg - 1) / tile_seg;
  float carry[VEC], r[VEC], h[VEC], u[SEG][VEC], fg[SEG][VEC], fx[SEG][VEC], d[SEG][VEC], A[VEC], Q[VEC];
  get_state<VEC>(a.dstate_out, b, a.D, ch, carry);
  for (int64_t q = p.nchunk - 1; q > chunk; q--)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const float2 m = p.agg[(q * a.B + b) * a.D + ch + i];
      carry[i] = map_s(m.x, carry[i], m.y);
    }
  int turn = 0;
  for (int64_t k = tiles - 1; k >= 0; k--, turn ^= 1) {
    const int64_t g = seg0 + k * tile_seg + w * TS + ts, t0 = g * SEG;
    const int nrow = g < seg1 ? (int)clamp64(a.T - t0, 0, SEG) : 0, n = g < seg1 ? (int)clamp64(len - t0, 0, SEG) : 0;
    get_state<VEC>(n > 0 ? a.record + g * a.D : nullptr, b, p.nseg * a.D, ch, h);
    const uint32_t keep = keep_bits(a, b, t0, n);
    load_backward<DT, VEC, TANH>(a, b, t0, ch, n, keep, h, u, fg, fx, d);
    segment_map_rev<VEC>(u, d, keep, A, Q);
    tile_scan<VEC, true>(lds[turn], nw, w, ts, cl, A, Q, carry, r);
    replay_rev<DT, VEC>(a, b, t0, ch, chan, n, nrow, keep, u, fg, fx, d, r);
  }
  if (w == 0 && ts == 0 && chan && a.dstate_in && chunk == 0) ops_st<HIERTCN_FP32, VEC>(a.dstate_in, b * a.D + ch, carry);
}

// the chunks' maps of the backward recurrence (gates and dout only)
template <int DT, int VEC>
__global__ __launch_bounds__(1024) void k_glr_agg_bwd(GlrP p) {
  constexpr int CL = CB / VEC, TS = 64 / CL;
  __shared__ float2 lds[2][16 * CB];
  const hiertcn_glr_t& a = p.a;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6, ts = lane / CL, cl = lane % CL;
  const int64_t blk = blockIdx.x, cb = blk % p.ncb, b = blk / p.ncb % a.B, chunk = blk / p.ncb / a.B;
  const bool chan = cb * CB + cl * VEC < a.D;
  const int64_t ch = chan ? cb * CB + cl * VEC : 0;
  const int64_t len = length_of(a, b);
  const int tile_seg = nw * TS;
  const int64_t seg0 = chunk * p.chunk_tiles * tile_seg;
  const int64_t seg1 = chunk + 1 < p.nchunk ? seg0 + (int64_t)p.chunk_tiles * tile_seg : p.nseg;
  const int64_t live = seg1 * SEG < len ? seg1 : (len + SEG - 1) / SEG;      // segments behind the end are identities
  const int64_t tiles = live > seg0 ? (live - seg0 + tile_seg - 1) / tile_seg : 0;
  float carry[VEC], carryA[VEC], none[VEC], u[SEG][VEC], d[SEG][VEC], A[VEC], Q[VEC];
#pragma unroll
  for (int i = 0; i < VEC; i++) carry[i] = 0.f, carryA[i] = 1.f;
  int turn = 0;
  for (int64_t k = tiles - 1; k >= 0; k--, turn ^= 1) {
    const int64_t g = seg0 + k * tile_seg + w * TS + ts, t0 = g * SEG;
    const int n = g < seg1 ? (int)clamp64(len - t0, 0, SEG) : 0;
    if (n > 0) {
      load_rows<DT, VEC>(a.gate, b * a.gate_sb + t0 * a.gate_st + ch, a.gate_st, n, u);
      load_rows<DT, VEC>(a.dout, b * a.dout_sb + t0 * a.dout_st + ch, a.dout_st, n, d);
    }
#pragma unroll
    for (int j = 0; j < SEG; j++)
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        float wv;
        if (j < n) gate_of(u[j][i], u[j][i], wv);
        else u[j][i] = 1.f, d[j][i] = 0.f;
      }
    segment_map_rev<VEC>(u, d, keep_bits(a, b, t0, n), A, Q);
    tile_scan<VEC, true>(lds[turn], nw, w, ts, cl, A, Q, carry, none);
    for (int q = 0; q < nw; q++)
#pragma unroll
      for (int i = 0; i < VEC; i++) carryA[i] = map_a(carryA[i], lds[turn][q * CB + cl * VEC + i].x);
  }
  if (w == 0 && ts == 0 && chan)
#pragma unroll
    for (int i = 0; i < VEC; i++) p.agg[(chunk * a.B + b) * a.D + ch + i] = make_float2(carryA[i], carry[i]);
}

// ---- launch selection --------------------------------------------------------------------------------------------------------------------------------
struct Plan { bool seq; int nw, nchunk, chunk_tiles; int64_t ncb; };

// vec: channels of a thread (1 where the width, a stride or an address is odd)
Plan plan_of(int64_t B, int64_t T, int64_t D, int vec, int most_waves) {
  Plan q{};
  const int ts = vec;                          // segments of a wave: 64 lanes / (64 channels / vec)
  const int64_t nseg = (T + SEG - 1) / SEG;
  q.ncb = (D + CB - 1) / CB;
  const int64_t seq_waves = (B * ((D + vec - 1) / vec) + 63) / 64;
  q.seq = nseg <= 1 || seq_waves >= 4096;
  q.nw = (int)((nseg + ts - 1) / ts < most_waves ? (nseg + ts - 1) / ts : most_waves);
  if (q.nw < 1) q.nw = 1;
  const int64_t tiles = (nseg + (int64_t)q.nw * ts - 1) / ((int64_t)q.nw * ts), wgs = B * q.ncb;
  int64_t want = wgs >= 512 ? 1 : (1024 + wgs - 1) / wgs;
  if (want > 64) want = 64;
  if (want > tiles) want = tiles;
  if (want < 1) want = 1;
  q.chunk_tiles = (int)((tiles + want - 1) / want);
  q.nchunk = (int)((tiles + q.chunk_tiles - 1) / q.chunk_tiles);
  if (q.nchunk < 1) q.nchunk = 1;
  return q;
}
constexpr int FWD_WAVES = 16, BWD_WAVES = 16;

size_t workspace_of(int64_t B, int64_t T, int64_t D) {
  size_t most = 0;
  for (int vec = 1; vec <= 2; vec++)
    for (int waves : {FWD_WAVES, BWD_WAVES}) {
      const Plan q = plan_of(B, T, D, vec, waves);
      const size_t need = q.seq || q.nchunk == 1 ? 0 : (size_t)(q.nchunk * B * D) * sizeof(float2) + (size_t)(B * D) * sizeof(float);
      if (need > most) most = need;
    }
  return most;
}

int check_shape(const hiertcn_glr_t* a) {
  if (!a) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  if (a->B < 0 || a->T < 0 || a->D < 0) return ops_fail(HIERTCN_ERR_INVALID, "negative size");
  if (a->B > (1ll << 31) || a->T > (1ll << 31) || a->D > (1ll << 31) || (a->B && a->D && a->B * a->D > (1ll << 40)))
    return ops_fail(HIERTCN_ERR_INVALID, "B, T, D are at most 2^31, B * D at most 2^40");
  if (!ops_dtype_ok(a->dtype)) return ops_fail(HIERTCN_ERR_INVALID, "dtype %d: 0 fp32, 1 bf16, 2 fp16", a->dtype);
  if (a->cand_act != 0 && a->cand_act != 1) return ops_fail(HIERTCN_ERR_INVALID, "cand_act %d: 0 none, 1 tanh", a->cand_act);
  return HIERTCN_OK;
}

// all addresses and strides of an operand allow `vec` elements at a time
bool aligned(const void* p, int64_t sb, int64_t st, int es, int vec) { return !p || ((uintptr_t)p % (size_t)(es * vec) == 0 && sb % vec == 0 && st % vec == 0); }

template <int DT, int VEC, bool TANH>
hipError_t go_forward(GlrP& p, const Plan& q, hipStream_t st) {
  const hiertcn_glr_t& a = p.a;
  if (q.seq) {
    const int64_t threads = a.B * (a.D / VEC);
    hipLaunchKernelGGL((k_glr_seq<DT, VEC, TANH>), dim3((unsigned)((threads + 63) / 64)), dim3(64), 0, st, p);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)(q.ncb * a.B * q.nchunk)), block(64 * q.nw);
  if (q.nchunk > 1) {
    hipLaunchKernelGGL((k_glr_tile<DT, VEC, TANH, true>), grid, block, 0, st, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((k_glr_tile<DT, VEC, TANH, false>), grid, block, 0, st, p);
  return hipGetLastError();
}
template <int DT, int VEC, bool TANH>
hipError_t go_backward(GlrP& p, const Plan& q, hipStream_t st) {
  const hiertcn_glr_t& a = p.a;
  if (q.seq) {
    const int64_t threads = a.B * (a.D / VEC);
    hipLaunchKernelGGL((k_glr_seq_bwd<DT, VEC, TANH>), dim3((unsigned)((threads + 63) / 64)), dim3(64), 0, st, p);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)(q.ncb * a.B * q.nchunk)), block(64 * q.nw);
  if (q.nchunk > 1) {
    hipLaunchKernelGGL((k_glr_agg_bwd<DT, VEC>), grid, block, 0, st, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((k_glr_tile_bwd<DT, VEC, TANH>), grid, block, 0, st, p);
  return hipGetLastError();
}
template <int VEC>
hipError_t go(GlrP& p, const Plan& q, bool backward, hipStream_t st) {
#define GLR_GO(DT)                                                                                                                   \
  return backward ? (p.a.cand_act ? go_backward<DT, VEC, true>(p, q, st) : go_backward<DT, VEC, false>(p, q, st))                     \
                  : (p.a.cand_act ? go_forward<DT, VEC, true>(p, q, st) : go_forward<DT, VEC, false>(p, q, st))
  switch (p.a.dtype) {
    case HIERTCN_FP32: GLR_GO(HIERTCN_FP32);
    case HIERTCN_BF16: GLR_GO(HIERTCN_BF16);
    default: GLR_GO(HIERTCN_FP16);
  }
#undef GLR_GO
}

int glr(const hiertcn_glr_t* in, bool backward, hipStream_t st) {
  if (int rc = check_shape(in)) return rc;
  GlrP p{};
  p.a = *in;
  hiertcn_glr_t& a = p.a;
  const int es = ops_size(a.dtype);
  if (a.B == 0 || a.D == 0) return HIERTCN_OK;
  if (a.T > 0 && (!a.gate || !a.cand || (backward ? !a.dout || !a.dgate || !a.dcand || !a.record : !a.out)))
    return ops_fail(HIERTCN_ERR_INVALID, "null gate, cand, %s", backward ? "dout, dgate, dcand or record" : "out");
  if (a.T == 0) {      // the state passes
    const float* src = backward ? a.dstate_out : a.state_in;
    float* dst = backward ? a.dstate_in : a.state_out;
    if (!dst || dst == src) return HIERTCN_OK;
    if (!src) return ops_fail(HIERTCN_ERR_INVALID, "T = 0 needs the state it passes on");
    OPS_TRY(hipMemcpyAsync(dst, src, (size_t)(a.B * a.D) * sizeof(float), hipMemcpyDeviceToDevice, st));
    return HIERTCN_OK;
  }
  for (int64_t* s : {&a.gate_sb, &a.cand_sb, &a.mask_sb, &a.out_sb, &a.dout_sb, &a.dgate_sb, &a.dcand_sb})
    if (a.B == 1) *s = 0;                   // the stride of a dimension of one is never taken
  for (int64_t* s : {&a.gate_st, &a.cand_st, &a.mask_st, &a.out_st, &a.dout_st, &a.dgate_st, &a.dcand_st})
    if (a.T == 1) *s = 0;
  for (int64_t s : {a.gate_sb, a.gate_st, a.cand_sb, a.cand_st, a.mask_sb, a.mask_st, a.out_sb, a.out_st, a.dout_sb, a.dout_st, a.dgate_sb, a.dgate_st, a.dcand_sb, a.dcand_st})
    if (s < 0 || s > (1ll << 50)) return ops_fail(HIERTCN_ERR_INVALID, "stride %lld", (long long)s);
  auto view = [&](const void* q, int64_t sb, int64_t s_t) { return OpsView{static_cast<const char*>(q), a.B, a.T, a.D, sb, s_t, es}; };
  const int64_t nseg = (a.T + SEG - 1) / SEG;
  const OpsView gate = view(a.gate, a.gate_sb, a.gate_st), cand = view(a.cand, a.cand_sb, a.cand_st);
  const OpsView mask{reinterpret_cast<const char*>(a.mask), a.B, a.T, 1, a.mask_sb, a.mask_st, 4}, lens = ops_flat(a.lengths, a.B, 4);
  const OpsView rec = ops_flat(a.record, a.B * nseg * a.D, 4), ws = ops_flat(a.workspace, (int64_t)(a.workspace ? a.workspace_bytes : 0), 1);
  OpsView ins[7] = {gate, cand, mask, lens}, outs[5];
  int ni = 4, no = 0;
  if (backward) {
    ins[ni++] = view(a.dout, a.dout_sb, a.dout_st);
    ins[ni++] = rec;
    ins[ni++] = ops_flat(a.dstate_out, a.B * a.D, 4);
    outs[no++] = view(a.dgate, a.dgate_sb, a.dgate_st);
    outs[no++] = view(a.dcand, a.dcand_sb, a.dcand_st);
    outs[no++] = ops_flat(a.dstate_in, a.B * a.D, 4);
  } else {
    if (a.state_in != a.state_out) ins[ni++] = ops_flat(a.state_in, a.B * a.D, 4);
    outs[no++] = view(a.out, a.out_sb, a.out_st);
    outs[no++] = rec;
    outs[no++] = ops_flat(a.state_out, a.B * a.D, 4);
  }
  outs[no++] = ws;
  for (int i = 0; i < no; i++) {
    if (outs[i].p && !ops_rows_apart(outs[i])) return ops_fail(HIERTCN_ERR_INVALID, "an output's rows overlap one another");
    for (int j = 0; j < ni; j++)
      if (ops_overlap(outs[i], ins[j])) return ops_fail(HIERTCN_ERR_INVALID, "an output overlaps an input");
    for (int j = i + 1; j < no; j++)
      if (ops_overlap(outs[i], outs[j])) return ops_fail(HIERTCN_ERR_INVALID, "two outputs overlap");
  }
  const void* f32[] = {a.mask, a.lengths, a.state_in, a.state_out, a.record, a.dstate_out, a.dstate_in};
  for (const void* q : f32)
    if ((uintptr_t)q % 4) return ops_fail(HIERTCN_ERR_INVALID, "an fp32 / int32 pointer is not a multiple of 4");
  for (const void* q : {a.gate, a.cand, (const void*)a.out, a.dout, (const void*)a.dgate, (const void*)a.dcand})
    if ((uintptr_t)q % (size_t)es) return ops_fail(HIERTCN_ERR_INVALID, "a pointer is not a multiple of its element");
  int vec = a.D % 2 == 0 ? 2 : 1;
  for (const void* q : f32)
    if ((uintptr_t)q % 8 && q != a.mask && q != a.lengths) vec = 1;
  if (!aligned(a.gate, a.gate_sb, a.gate_st, es, vec) || !aligned(a.cand, a.cand_sb, a.cand_st, es, vec) || !aligned(a.out, a.out_sb, a.out_st, es, vec) ||
      !aligned(a.dout, a.dout_sb, a.dout_st, es, vec) || !aligned(a.dgate, a.dgate_sb, a.dgate_st, es, vec) || !aligned(a.dcand, a.dcand_sb, a.dcand_st, es, vec))
    vec = 1;
  const Plan q = plan_of(a.B, a.T, a.D, vec, backward ? BWD_WAVES : FWD_WAVES);
  p.nseg = nseg;
  p.ncb = (int)q.ncb;
  p.nchunk = q.nchunk;
  p.chunk_tiles = q.chunk_tiles;
  if (!q.seq && q.nchunk > 1) {
    const size_t need = workspace_of(a.B, a.T, a.D);      // (the most that any alignment and direction takes)
    if (!a.workspace || a.workspace_bytes < need || (uintptr_t)a.workspace % 16)
      return ops_fail(HIERTCN_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", need, a.workspace ? a.workspace_bytes : (size_t)0);
    p.agg = static_cast<float2*>(a.workspace);
    p.state0 = reinterpret_cast<float*>(p.agg + q.nchunk * a.B * a.D);
  }
  const int64_t blocks = q.seq ? (a.B * ((a.D + vec - 1) / vec) + 63) / 64 : q.ncb * a.B * q.nchunk;
  if (blocks > 0x7fffffffll) return ops_fail(HIERTCN_ERR_INVALID, "B * D is too large for one launch");
  OPS_TRY(vec == 2 ? go<2>(p, q, backward, st) : go<1>(p, q, backward, st));
  return HIERTCN_OK;
}

}  // namespace

extern "C" {

size_t hiertcn_glr_record_floats(int64_t B, int64_t T, int64_t D) { return B > 0 && T > 0 && D > 0 ? (size_t)(B * ((T + SEG - 1) / SEG) * D) : 0; }
size_t hiertcn_glr_workspace_bytes(int64_t B, int64_t T, int64_t D) { return B > 0 && T > 0 && D > 0 ? workspace_of(B, T, D) : 0; }
int hiertcn_glr_forward(const hiertcn_glr_t* a, void* stream) { return glr(a, false, reinterpret_cast<hipStream_t>(stream)); }
int hiertcn_glr_backward(const hiertcn_glr_t* a, void* stream) { return glr(a, true, reinterpret_cast<hipStream_t>(stream)); }

}  // extern "C"
