// Gated linear recurrence (include/hiertcn_ops.h): h_t = u_t [keep_t] h_{t-1} + (1 - u_t) c_t with u = sigmoid(gate) and c = cand or tanh(cand) --
// the update of customed_gru_cell.py:309-337 with gates that do not read the state, hence a scan.
//
// The map of a run of steps is h -> A h + S (A the product of the a_t = u_t keep_t, S the run's own state from zero), and maps compose:
// (A2, S2) after (A1, S1) is (A2 A1, A2 S1 + S2).  Time is cut into SEGMENTS of 16 steps.  A wave owns a segment of 64 VEC neighbouring channels of one
// sequence, so that everything but the channels -- rows, masks, lengths, branches -- is uniform over it and lives in scalar registers.  It keeps its
// a_t and (1 - u_t) c_t in vector registers, so that gate and cand are read once: it forms (A, S), learns the state before its segment from the
// maps of the segments before it (waves of the workgroup, a TILE, through LDS; earlier tiles as a carry in registers), and replays the segment from there.
//
// Where there are few sequences for the machine the tiles of a sequence go to different workgroups (CHAIN).  A workgroup publishes its tile's map, applies
// those of the tiles before it in its group of 16 to the state before the group, and the last of a group publishes the state behind it.  The order of
// all that is the order of time, whoever waits for whom, so results do not depend on timing.  A word (A, S) is its own flag: 64 bits, written by one store that
// goes past the L2s, all ones until then (a NaN is stored as the canonical one, so that no result looks like that).  A workgroup takes the tile of its TICKET, drawn
// when it starts, and waits for lower tickets only: those run, and the lowest waits for nobody, so every wait ends, however workgroups are dispatched.  Should a
// word never come all the same (a workspace that two calls use at once), its waits give up after some seconds: what could not be learnt is NaN and the launch ends.
//
// The backward pass is the same recurrence the other way round, lambda_t = dout_t + a_{t+1} lambda_{t+1}: with r_t = a_t lambda_t a run maps r -> A r + Q
// with the same A.  States are not read back from the rounded output: the forward pass leaves the fp32 state before every segment in `record`, 1/16 of
// a [B][T][D] fp32 array, and a wave replays its segment from there.
//
// Bound by memory where the arrays are large and by the latency of a tile (load, fold, replay, store) where they are not: 8.9 / 12.5 us forward / backward at
// 32 x 200 x 128 fp32, 18.0 / 25.8 at 64 x 500 x 256 bf16, 92 / 159 (4.2 TB/s) at 512 x 500 x 256 bf16, 115 / 199 (3.5 / 3.4 TB/s, half of the cycles in vector
// instructions) at 2 x 65536 x 512 bf16 chained, 94 / 137 (4.2 / 4.8 TB/s) at 128 x 2000 x 128 fp32; a copy of many GB runs at 4.8.  A single step of 32 x 256: 4.8 us,
// a launch.  Fetching the next tile before the fold of this one costs registers and waves: 114 -> 155 chained, nothing gained elsewhere.
//
// A reset has to cut a state that is NaN or infinite (0 * NaN = NaN), and nothing else may: A is exactly 0 only where a reset lies in the run, and a map with A = 0
// ignores what it is applied to.  The product of the gates alone is kept from underflowing to 0: an infinite state stays infinite however many gates are all but
// shut (0 * inf = NaN).  Without a mask maps are plain fma's.
#include "ops.h"

#ifdef HIERTCN_TEST_HOOKS
#include <stdlib.h>
#endif

namespace {

constexpr int SEG = 16;          // steps of a segment = distance of the records
constexpr int MAXW = 16;         // waves of a workgroup, at most
constexpr float TINY = 1.401298464e-45f;

struct GlrP {
  hiertcn_glr_t a;
  int nseg;                      // ceil(T / SEG)
  int ncb;                       // channel blocks
  // CHAIN
  int ntile;                     // tiles of a sequence, each a workgroup
  uint64_t* map;                 // [ntile][B][D]: the tiles' maps
  uint64_t* behind;              // [ntile / GROUP][B][D]: the state behind a group, in the low half
  float* state0;                 // [B][D]: the state before the first tile (state_out may be state_in)
  unsigned* ticket;              // and, behind it, whether a wait has given up
  unsigned grid, polls;          // workgroups; looks of a wait
};
constexpr int GROUP = 16;        // tiles of a group

// maps: composition and application.  CUT: A = 0 marks a reset
template <bool CUT>
__device__ __forceinline__ float map_a(float A1, float A2) { return !CUT ? fmaxf(A1 * A2, TINY) : A1 == 0.f || A2 == 0.f ? 0.f : fmaxf(A1 * A2, TINY); }
template <bool CUT>
__device__ __forceinline__ float map_s(float A2, float S1, float S2) { return CUT && A2 == 0.f ? S2 : fmaf(A2, S1, S2); }

// (The exponential of 16-bit operands is |x| half steps of fp32 off, 2^-13 or less of the operand's own: 4096 x 30 x 256 bf16 43 / 71 us, 49 / 77 with the better one.)
// u = sigmoid(g) and w = 1 - u = sigmoid(-g), each to 8 half steps and what the exponential adds (1 - u formed from u would lose the small ones)
template <int DT>
__device__ __forceinline__ void gate_of(float g, float& u, float& w) {
  const float e = ops_exp_of<DT>(-fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
  u = g >= 0.f ? r : er;
  w = g >= 0.f ? er : r;
}
// tanh to as much: the odd series where (1 - e^-2x) / (1 + e^-2x) would cancel; and its slope 4 e^-2x / (1 + e^-2x)^2 (1 - tanh^2, formed from a rounded tanh, is
// all error from |x| = 8 on)
template <int DT>
__device__ __forceinline__ float tanh_of(float x, float& slope) {
  const float a = fabsf(x), x2 = x * x;
  const float e = ops_exp_of<DT>(-2.f * a);
  const float r = __builtin_amdgcn_rcpf(1.f + e);
  const float big = copysignf((1.f - e) * r, x);
  slope = 4.f * e * r * r;
  float s = fmaf(x2, -8.863235530e-3f, 2.186948854e-2f);     // x - x^3/3 + 2x^5/15 - 17x^7/315 + 62x^9/2835 - 1382x^11/155925
  s = fmaf(x2, s, -5.396825397e-2f);
  s = fmaf(x2, s, 1.333333333e-1f);
  s = fmaf(x2, s, -3.333333333e-1f);
  return a < 0.3f ? fmaf(x * x2, s, x) : big;
}

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
// steps of a sequence that count, as a scalar (a load through a pointer that the outputs might alias is not one by itself)
__device__ __forceinline__ int length_of(const hiertcn_glr_t& a, int64_t b) {
  return __builtin_amdgcn_readfirstlane(a.lengths ? clamped(a.lengths[b], 0, (int)a.T) : (int)a.T);
}

// The mask of the steps t0 .. t0 + n - 1 (n >= 1), one to a lane; and the uniform word whose bit j says whether step t0 + j keeps the state (steps behind the end do)
template <bool CUT>
__device__ __forceinline__ float load_mask(const hiertcn_glr_t& a, int64_t b, int t0, int n) {
  const int lane = threadIdx.x & 63;
  return CUT ? a.mask[b * a.mask_sb + (t0 + (lane < n ? lane : n - 1)) * a.mask_st] : 1.f;
}
template <bool CUT>
__device__ __forceinline__ uint32_t keep_bits(float mask, int n) {
  return CUT ? ~(uint32_t)__ballot((int)(threadIdx.x & 63) < n && mask == 0.f) : 0xffffffffu;
}
// x, or 0 where bit j of the (uniform) word is clear: an AND with 0 or all ones, which takes NaN and infinity too
template <bool CUT>
__device__ __forceinline__ float held(float x, uint32_t keep, int j) {
  return CUT ? __builtin_bit_cast(float, __builtin_bit_cast(int, x) & __builtin_amdgcn_sbfe((int)keep, j, 1)) : x;
}
// The word again, opaque to the optimiser: the 16 masks that it stands for are formed anew in every loop instead of living in scalar registers throughout.
__device__ __forceinline__ uint32_t anew(uint32_t keep) {
  asm volatile("" : "+s"(keep));
  return keep;
}
// A wave's place: everything here but `off` and `chan` is uniform.
template <int VEC>
struct Place {
  int w, nw, off;                // wave of the workgroup, waves; this lane's first channel of the block
  int tile;                      // CHAIN's, in the order of the tickets
  int64_t b, ch0;
  bool chan;
  __device__ Place(const GlrP& p, unsigned blk) {
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    nw = blockDim.x >> 6;
    const unsigned per = (unsigned)p.ncb * (unsigned)p.a.B;      // (the grid fits 31 bits)
    tile = (int)(blk / per);
    const unsigned rest = blk % per;
    b = rest / (unsigned)p.ncb;
    ch0 = (int64_t)(rest % (unsigned)p.ncb) * 64 * VEC;
    off = (threadIdx.x & 63) * VEC;
    chan = ch0 + off < p.a.D;
    if (!chan) off = 0;
  }
};
// a [.][D] fp32 row of states
template <int VEC>
__device__ __forceinline__ void get_state(const float* p, int64_t row, const Place<VEC>& at, float (&h)[VEC]) {
  if (p) ops_ld<HIERTCN_FP32, VEC>(p + row, at.off, h);
  else
#pragma unroll
    for (int i = 0; i < VEC; i++) h[i] = 0.f;
}
template <int VEC>
__device__ __forceinline__ void put_state(float* p, int64_t row, const Place<VEC>& at, const float (&h)[VEC]) {
  if (at.chan) ops_st<HIERTCN_FP32, VEC>(p + row, at.off, h);
}
template <int DT>
__device__ __forceinline__ const char* row_ptr(const void* p, int64_t off) { return static_cast<const char*>(p) + off * (DT == HIERTCN_FP32 ? 4 : 2); }

// The n >= 1 live rows of a segment; a dead step reads the last live row again (no branches: all loads are in flight together).
template <int DT, int VEC>
__device__ __forceinline__ void load_rows(const void* p, int64_t base, int64_t st, int off, int n, typename OpsRaw<DT, VEC>::type (&o)[SEG]) {
  const char* q = row_ptr<DT>(p, base);
#pragma unroll
  for (int j = 0; j < SEG; j++) {
    o[j] = reinterpret_cast<const typename OpsRaw<DT, VEC>::type*>(q)[off / VEC];
    q = row_ptr<DT>(q, j + 1 < n ? st : 0);
  }
}

// the first nrow rows of a segment
template <int DT, int VEC>
__device__ __forceinline__ void store_rows(const char* q, int64_t st, const Place<VEC>& at, int nrow, const float (&o)[SEG][VEC]) {
  if (nrow == SEG) {
    if (at.chan)
#pragma unroll
      for (int j = 0; j < SEG; j++, q = row_ptr<DT>(q, st)) ops_st<DT, VEC>(const_cast<char*>(q), at.off, o[j]);
  } else if (at.chan) {
#pragma unroll
    for (int j = 0; j < SEG; j++, q = row_ptr<DT>(q, st))
      if (j < nrow) ops_st<DT, VEC>(const_cast<char*>(q), at.off, o[j]);
  }
}

// the product of a segment's gates as the A of its map
template <int VEC, bool CUT>
__device__ __forceinline__ void close_map(uint32_t keep, float (&A)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i++) A[i] = !CUT || keep == 0xffffffffu ? (A[i] < TINY ? TINY : A[i]) : 0.f;      // (a NaN stays)
}

// The state before (REV: behind) every wave's segment, given `carry` before the tile; `carry` behind it.  One barrier; `lds` alternates between two buffers, so
// that the next tile's writes need no second one.
template <int VEC>
__device__ __forceinline__ void put_map(float2* lds, const Place<VEC>& at, const float (&A)[VEC], const float (&S)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; i++) lds[(at.w * VEC + i) * 64 + (threadIdx.x & 63)] = make_float2(A[i], S[i]);
}
// folds the maps of the waves onto `carry`, in the order of time; h: before this wave's
template <int VEC, bool CUT, bool REV>
__device__ __forceinline__ void fold_waves(const float2* lds, const Place<VEC>& at, float (&carry)[VEC], float (&h)[VEC]) {
  const int lane = threadIdx.x & 63;
  for (int q0 = 0; q0 < at.nw; q0 += 4) {
    float2 m[4][VEC];
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const int q = q0 + k < at.nw ? q0 + k : at.nw - 1;
        m[k][i] = lds[((REV ? at.nw - 1 - q : q) * VEC + i) * 64 + lane];
      }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (q0 + k >= at.nw) break;
      if ((REV ? at.nw - 1 - (q0 + k) : q0 + k) == at.w)
#pragma unroll
        for (int i = 0; i < VEC; i++) h[i] = carry[i];
#pragma unroll
      for (int i = 0; i < VEC; i++) carry[i] = map_s<CUT>(m[k][i].x, carry[i], m[k][i].y);
    }
  }
}
template <int VEC, bool CUT, bool REV>
__device__ __forceinline__ void tile_scan(float2* lds, const Place<VEC>& at, const float (&A)[VEC], const float (&S)[VEC], float (&carry)[VEC], float (&h)[VEC]) {
  if (at.nw == 1) {
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      h[i] = carry[i];
      carry[i] = map_s<CUT>(A[i], carry[i], S[i]);
    }
    return;
  }
  put_map<VEC>(lds, at, A, S);
  __syncthreads();
  fold_waves<VEC, CUT, REV>(lds, at, carry, h);
}

#ifdef HIERTCN_TEST_HOOKS       // the test of the waits' bound: a launch whose words never come (GlrP's polls from the environment).  In no shipped library.
#define GLR_PUBLISH (p.polls == OPS_POLLS)
#else
#define GLR_PUBLISH true
#endif
// ---- CHAIN ------------------------------------------------------------------------------------------------------------------------------------------
// What a chained workgroup keeps in LDS: the maps of its waves, those of the tiles before it in its group, the state before the group, the ticket.
template <int VEC>
struct ChainLds {
  float2* waves;                 // [nw][VEC][64]
  float2* tiles;                 // [GROUP - 1][VEC][64]
  float* first;                  // [VEC][64]
  unsigned* ticket;
  __device__ explicit ChainLds(float2* lds) {
    waves = lds;
    tiles = waves + (blockDim.x >> 6) * VEC * 64;
    first = reinterpret_cast<float*>(tiles + (GROUP - 1) * VEC * 64);
    ticket = reinterpret_cast<unsigned*>(first + VEC * 64);
  }
  static size_t bytes(int nw) { return (size_t)(nw + GROUP - 1) * VEC * 64 * sizeof(float2) + VEC * 64 * sizeof(float) + 16; }
};
// tile_scan over workgroups: wave 0 publishes the tile's map, and every wave fetches its share of the words that the state before the tile is made of.
template <int VEC, bool CUT, bool REV>
__device__ __forceinline__ void chain_scan(const GlrP& p, const ChainLds<VEC>& lds, const Place<VEC>& at, const float (&A)[VEC], const float (&S)[VEC], float (&carry)[VEC],
                                           float (&h)[VEC]) {
  const int lane = threadIdx.x & 63, place = at.tile % GROUP, group = at.tile / GROUP;
  const int64_t plane = p.a.B * p.a.D, row = at.b * p.a.D + at.ch0;
  float tA[VEC], tS[VEC];
#pragma unroll
  for (int i = 0; i < VEC; i++) tA[i] = 1.f, tS[i] = 0.f;
  put_map<VEC>(lds.waves, at, A, S);
  __syncthreads();
  if (at.w == 0 && at.tile + 1 < p.ntile) {
    float none[VEC];
    fold_waves<VEC, CUT, REV>(lds.waves, at, tS, none);
    for (int q = 0; q < at.nw; q++)
#pragma unroll
      for (int i = 0; i < VEC; i++) tA[i] = map_a<CUT>(tA[i], lds.waves[(q * VEC + i) * 64 + lane].x);
    if (GLR_PUBLISH && at.chan && place + 1 < GROUP)
#pragma unroll
      for (int i = 0; i < VEC; i++) ops_publish(p.map + (int64_t)at.tile * plane + row + at.off + i, ops_word(tS[i], tA[i]));
  }
  for (int q = at.w; q < place; q += at.nw)
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const uint64_t v = ops_await(p.map + (int64_t)(group * GROUP + q) * plane + row + at.off + i, p.ticket + 1, p.polls);
      lds.tiles[(q * VEC + i) * 64 + lane] = make_float2(ops_high(v), ops_low(v));
    }
  if (at.w == at.nw - 1) {
    float f[VEC];
    if (group == 0) get_state<VEC>(p.state0, row, at, f);
#pragma unroll
    for (int i = 0; i < VEC; i++) lds.first[i * 64 + lane] = group == 0 ? f[i] : ops_low(ops_await(p.behind + (int64_t)(group - 1) * plane + row + at.off + i, p.ticket + 1, p.polls));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VEC; i++) carry[i] = lds.first[i * 64 + lane];
  for (int q0 = 0; q0 < place; q0 += 4) {
    float2 m[4][VEC];
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int i = 0; i < VEC; i++) m[k][i] = lds.tiles[((q0 + k < place ? q0 + k : q0) * VEC + i) * 64 + lane];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (q0 + k < place)
#pragma unroll
        for (int i = 0; i < VEC; i++) carry[i] = map_s<CUT>(m[k][i].x, carry[i], m[k][i].y);
  }
  if (GLR_PUBLISH && at.w == 0 && at.chan && place + 1 == GROUP && at.tile + 1 < p.ntile)
#pragma unroll
    for (int i = 0; i < VEC; i++) ops_publish(p.behind + (int64_t)group * plane + row + at.off + i, ops_word(map_s<CUT>(tA[i], carry[i], tS[i]), 0.f));
  fold_waves<VEC, CUT, REV>(lds.waves, at, carry, h);
}
// clears what a chain's words start from
__global__ __launch_bounds__(256) void k_chain_init(GlrP p, const float* first, int64_t words) {
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, n = p.a.B * p.a.D;
  if (i0 < 2) p.ticket[i0] = 0;
  for (int64_t i = i0; i < words; i += (int64_t)gridDim.x * 256) p.map[i] = OPS_NOTHING;
  for (int64_t i = i0; i < n; i += (int64_t)gridDim.x * 256) p.state0[i] = first ? first[i] : 0.f;
}

// ---- forward: a workgroup takes 64 VEC channels of one sequence through time, nw segments (a tile) at a time; CHAIN: one tile ---------------------------
template <int DT, int VEC, bool TANH, bool CUT, bool CHAIN>
__global__ __launch_bounds__(64 * MAXW / VEC) void k_glr(GlrP p) {
  extern __shared__ float2 lds[];          // 2 x [nw][VEC][64]; CHAIN: ChainLds
  const hiertcn_glr_t& a = p.a;
  const ChainLds<VEC> chain(lds);
  const unsigned blk = CHAIN ? ops_ticket(p.ticket, chain.ticket) : blockIdx.x;
  if (CHAIN && blk >= p.grid) return;      // (never, but with a workspace that two calls use at once)
  const Place<VEC> at(p, blk);
  const int64_t row = at.b * a.D + at.ch0;
  const int len = length_of(a, at.b), seg0 = CHAIN ? at.tile * at.nw : 0, seg1 = CHAIN && seg0 + at.nw < p.nseg ? seg0 + at.nw : p.nseg;
  float carry[VEC], h[VEC], u[SEG][VEC], s[SEG][VEC], A[VEC], S[VEC];
  typename OpsRaw<DT, VEC>::type rg[SEG], rc[SEG];
  if (!CHAIN) get_state<VEC>(a.state_in, row, at, carry);
  int turn = 0;
  for (int g0 = seg0; g0 < seg1; g0 += at.nw, turn ^= 1) {
    const int g = g0 + at.w, t0 = g * SEG, n = clamped(len - t0, 0, SEG), nrow = g < seg1 ? clamped((int)a.T - t0, 0, SEG) : 0;
    uint32_t keep = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < VEC; i++) A[i] = 1.f, S[i] = 0.f;
    if (n > 0) {
      const float mask = load_mask<CUT>(a, at.b, t0, n);
      load_rows<DT, VEC>(a.gate, at.b * a.gate_sb + t0 * a.gate_st + at.ch0, a.gate_st, at.off, n, rg);
      load_rows<DT, VEC>(a.cand, at.b * a.cand_sb + t0 * a.cand_st + at.ch0, a.cand_st, at.off, n, rc);
      __builtin_amdgcn_sched_barrier(0);
      keep = __builtin_amdgcn_readfirstlane(keep_bits<CUT>(mask, n));
#pragma unroll
      for (int j = 0; j < SEG; j++) {
        float g4[VEC], c4[VEC];
        ops_cvt<DT, VEC>(rg[j], g4);
        ops_cvt<DT, VEC>(rc[j], c4);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          float w;
          gate_of<DT>(g4[i], u[j][i], w);
          float slope;
          s[j][i] = w * (TANH ? tanh_of<DT>(c4[i], slope) : c4[i]);
        }
      }
      if (n < SEG)                         // dead steps: the identity
#pragma unroll
        for (int j = 1; j < SEG; j++)
#pragma unroll
          for (int i = 0; i < VEC; i++)
            if (j >= n) u[j][i] = 1.f, s[j][i] = 0.f;
#pragma unroll
      for (int j = 0; j < SEG; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          S[i] = fmaf(u[j][i], held<CUT>(S[i], keep, j), s[j][i]);
          A[i] *= u[j][i];
        }
      close_map<VEC, CUT>(keep, A);
    }
    if (CHAIN) chain_scan<VEC, CUT, false>(p, chain, at, A, S, carry, h);
    else tile_scan<VEC, CUT, false>(lds + turn * at.nw * VEC * 64, at, A, S, carry, h);
    if (a.record && nrow > 0) put_state<VEC>(a.record, (at.b * p.nseg + g) * a.D + at.ch0, at, h);
    if (CUT) keep = anew(keep);
    const char* o = row_ptr<DT>(a.out, at.b * a.out_sb + t0 * a.out_st + at.ch0);
    if (n > 0)
#pragma unroll
      for (int j = 0; j < SEG; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          h[i] = fmaf(u[j][i], held<CUT>(h[i], keep, j), s[j][i]);
          s[j][i] = j < n ? h[i] : 0.f;
        }
    else
#pragma unroll
      for (int j = 0; j < SEG; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) s[j][i] = 0.f;
    store_rows<DT, VEC>(o, a.out_st, at, nrow, s);
  }
  if (at.w == 0 && a.state_out && seg1 == p.nseg) put_state<VEC>(a.state_out, row, at, carry);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------------------------
// Per element: u, fg = (h_prev - c) u (1 - u) and fx = (1 - u) act'(c), so that dgate = lambda fg and dcand = lambda fx; d = dout.
// CHAIN: the tiles in the order of the tickets are the sequence's from its end.
template <int DT, int VEC, bool TANH, bool CUT, bool CHAIN>
__global__ __launch_bounds__(64 * MAXW) void k_glr_bwd(GlrP p) {
  extern __shared__ float2 lds[];          // as in k_glr
  const hiertcn_glr_t& a = p.a;
  const ChainLds<VEC> chain(lds);
  const unsigned blk = CHAIN ? ops_ticket(p.ticket, chain.ticket) : blockIdx.x;
  if (CHAIN && blk >= p.grid) return;      // (never, but with a workspace that two calls use at once)
  const Place<VEC> at(p, blk);
  const int64_t row = at.b * a.D + at.ch0;
  const int len = length_of(a, at.b), seg0 = CHAIN ? (p.ntile - 1 - at.tile) * at.nw : 0, seg1 = CHAIN && seg0 + at.nw < p.nseg ? seg0 + at.nw : p.nseg;
  const int tiles = (seg1 - seg0 + at.nw - 1) / at.nw;
  float carry[VEC], r[VEC], h[VEC], u[SEG][VEC], fg[SEG][VEC], fx[SEG][VEC], d[SEG][VEC], A[VEC], Q[VEC];
  typename OpsRaw<DT, VEC>::type rg[SEG], rc[SEG], rd[SEG];
  if (!CHAIN) get_state<VEC>(a.dstate_out, row, at, carry);
  int turn = 0;
  for (int k = tiles - 1; k >= 0; k--, turn ^= 1) {
    const int g = seg0 + k * at.nw + at.w, t0 = g * SEG;
    const int nrow = g < seg1 ? clamped((int)a.T - t0, 0, SEG) : 0, n = g < seg1 ? clamped(len - t0, 0, SEG) : 0;
    uint32_t keep = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < VEC; i++) A[i] = 1.f, Q[i] = 0.f;
    if (n > 0) {
      const float mask = load_mask<CUT>(a, at.b, t0, n);
      get_state<VEC>(a.record, (at.b * p.nseg + g) * a.D + at.ch0, at, h);
      load_rows<DT, VEC>(a.gate, at.b * a.gate_sb + t0 * a.gate_st + at.ch0, a.gate_st, at.off, n, rg);
      load_rows<DT, VEC>(a.cand, at.b * a.cand_sb + t0 * a.cand_st + at.ch0, a.cand_st, at.off, n, rc);
      load_rows<DT, VEC>(a.dout, at.b * a.dout_sb + t0 * a.dout_st + at.ch0, a.dout_st, at.off, n, rd);
      __builtin_amdgcn_sched_barrier(0);
      keep = __builtin_amdgcn_readfirstlane(keep_bits<CUT>(mask, n));
#pragma unroll
      for (int j = 0; j < SEG; j++) {
        float g4[VEC], c4[VEC];
        ops_cvt<DT, VEC>(rg[j], g4);
        ops_cvt<DT, VEC>(rc[j], c4);
        ops_cvt<DT, VEC>(rd[j], d[j]);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          float w, slope = 1.f;
          gate_of<DT>(g4[i], u[j][i], w);
          const float c = TANH ? tanh_of<DT>(c4[i], slope) : c4[i];
          const float hp = held<CUT>(h[i], keep, j);
          h[i] = fmaf(u[j][i], hp, w * c);
          fg[j][i] = (hp - c) * (u[j][i] * w);
          fx[j][i] = w * slope;
        }
      }
      if (n < SEG)                         // dead steps: the identity, no gradient
#pragma unroll
        for (int j = 1; j < SEG; j++)
#pragma unroll
          for (int i = 0; i < VEC; i++)
            if (j >= n) u[j][i] = 1.f, fg[j][i] = fx[j][i] = d[j][i] = 0.f;
#pragma unroll
      for (int j = SEG - 1; j >= 0; j--)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          Q[i] = held<CUT>(u[j][i] * (d[j][i] + Q[i]), keep, j);
          A[i] *= u[j][i];
        }
      close_map<VEC, CUT>(keep, A);
    }
    if (CHAIN) chain_scan<VEC, CUT, true>(p, chain, at, A, Q, carry, r);
    else tile_scan<VEC, CUT, true>(lds + turn * at.nw * VEC * 64, at, A, Q, carry, r);
    if (CUT) keep = anew(keep);
    if (n > 0)
#pragma unroll
      for (int j = SEG - 1; j >= 0; j--)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const float lam = d[j][i] + r[i];
          fg[j][i] *= lam;                 // (a dead step has fg = fx = 0)
          fx[j][i] *= lam;
          r[i] = held<CUT>(u[j][i] * lam, keep, j);
        }
    else
#pragma unroll
      for (int j = 0; j < SEG; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) fg[j][i] = fx[j][i] = 0.f;
    store_rows<DT, VEC>(row_ptr<DT>(a.dgate, at.b * a.dgate_sb + t0 * a.dgate_st + at.ch0), a.dgate_st, at, nrow, fg);
    store_rows<DT, VEC>(row_ptr<DT>(a.dcand, at.b * a.dcand_sb + t0 * a.dcand_st + at.ch0), a.dcand_st, at, nrow, fx);
  }
  if (at.w == 0 && a.dstate_in && seg0 == 0) put_state<VEC>(a.dstate_in, row, at, carry);
}

// ---- launch selection --------------------------------------------------------------------------------------------------------------------------------
struct Plan { int vec, nw; bool chain; int64_t ncb, ntile; };

// wide: the width, every stride and every address allow two channels of a thread at a time.  Measured on (lanes x steps x width), us, forward / backward:
//   two channels where that still leaves 8 waves a SIMD: 512 x 500 x 256 bf16 95 against 119; else one, for the waves: 64 x 500 x 256 18.5 against 31
//   one workgroup through a sequence where there are 256 of them: 64 x 500 x 256 19 / 28 against 25 / 35 chained; chained where there are fewer:
//   2 x 65536 x 512 116 / 190 against 1670 / 2210, 8 x 500 x 256 12 / 14 against 16 / 23
//   waves of a workgroup: as few as make 4096 in all (4096 x 30 x 256 one: 49 / 76, two 65 / 130 before; 512 x 500 x 256 four: 95 / 153, eight 97 / 160); chained
//   eight (2 x 65536 x 512 132 / 189 against 160 / 215 with sixteen), but sixteen where 256 to 512 workgroups of sixteen make it all: the chain is half as long.  Sixteen
//   against eight, with k_chain_init: 17 x 1001 x 333 fp16 24.8 / 32.4 against 27.6 / 32.2, 8 x 1001 x 512 bf16 17.5 / 20.9 against 19.9 / 23.0, 4 x 4000 x 256 bf16
//   18.3 / 22.1 against 20.7 / 24.1, 2 x 20000 x 128 fp32 27.7 / 34.4 against 31.2 / 33.6, 40 x 700 x 200 fp32 26.3 / 36.6 against 29.5 / 34.5, 1 x 130000 x 64 bf16
//   46 / 49 against 82 / 80; the one loss of nine shapes 12 x 1500 x 256 fp32, 25.5 / 32.3 against 24.6 / 28.2.  (A compute unit holds one workgroup of sixteen waves of
//   75 to 107 registers, so up to 256 of them are resident and the others follow.)
Plan plan_of(int64_t B, int64_t T, int64_t D, bool wide, bool backward) {
  Plan q{};
  const int64_t nseg = (T + SEG - 1) / SEG;
  q.vec = wide && !backward && B * ((D + 127) / 128) * nseg >= 8192 ? 2 : 1;
  q.ncb = (D + 64 * q.vec - 1) / (64 * q.vec);
  const int64_t wgs = B * q.ncb, generation = wgs * ((nseg + MAXW - 1) / MAXW);
  q.chain = nseg > MAXW && wgs < 256;
  const int64_t waves = !q.chain ? (4096 + wgs - 1) / wgs : generation >= 256 && generation <= 512 ? MAXW : 8;
  const int most = MAXW / q.vec;               // (what the registers of a workgroup allow)
  q.nw = (int)(waves > most ? most : waves < 1 ? 1 : waves);
  if (q.nw > nseg) q.nw = (int)nseg;
  q.ntile = (nseg + q.nw - 1) / q.nw;
  return q;
}
int64_t words_of(const Plan& q, int64_t B, int64_t D) { return (q.ntile + q.ntile / GROUP + 1) * B * D; }
size_t bytes_of(const Plan& q, int64_t B, int64_t D) { return q.chain ? (size_t)words_of(q, B, D) * 8 + (size_t)(B * D) * 4 + 256 : 0; }

size_t workspace_of(int64_t B, int64_t T, int64_t D) {
  size_t most = 0;
  for (bool wide : {false, true})
    for (bool backward : {false, true}) {
      const size_t need = bytes_of(plan_of(B, T, D, wide, backward), B, D);
      if (need > most) most = need;
    }
  return most;
}

int check_shape(const hiertcn_glr_t* a) {
  if (!a) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  if (a->B < 0 || a->T < 0 || a->D < 0) return ops_fail(HIERTCN_ERR_INVALID, "negative size");
  if (a->B > (1ll << 31) || a->T >= (1ll << 31) - 1024 || a->D > (1ll << 31) || (a->B && a->D && a->B * a->D > (1ll << 40)))
    return ops_fail(HIERTCN_ERR_INVALID, "B and D are at most 2^31, T below 2^31 - 1024, B * D at most 2^40");
  if (!ops_dtype_ok(a->dtype)) return ops_fail(HIERTCN_ERR_INVALID, "dtype %d: 0 fp32, 1 bf16, 2 fp16", a->dtype);
  if (a->cand_act != 0 && a->cand_act != 1) return ops_fail(HIERTCN_ERR_INVALID, "cand_act %d: 0 none, 1 tanh", a->cand_act);
  return HIERTCN_OK;
}

// all addresses and strides of an operand allow `vec` elements at a time
bool aligned(const void* p, int64_t sb, int64_t st, int es, int vec) { return !p || ((uintptr_t)p % (size_t)(es * vec) == 0 && sb % vec == 0 && st % vec == 0); }

template <int DT, int VEC, bool TANH, bool CUT>
hipError_t go(const GlrP& p, const Plan& q, bool backward, hipStream_t st) {
  const dim3 grid((unsigned)(q.ncb * p.a.B * (q.chain ? q.ntile : 1))), block(64 * q.nw);
  const size_t maps = (size_t)q.nw * q.vec * 64 * sizeof(float2);
  if (q.chain) {
    const int64_t words = words_of(q, p.a.B, p.a.D);
    hipLaunchKernelGGL(k_chain_init, dim3((unsigned)(words / 1024 + 1 < 2048 ? words / 1024 + 1 : 2048)), dim3(256), 0, st, p, backward ? p.a.dstate_out : p.a.state_in, words);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const size_t lds = q.vec == 2 ? ChainLds<2>::bytes(q.nw) : ChainLds<1>::bytes(q.nw);
    if (backward) hipLaunchKernelGGL((k_glr_bwd<DT, 1, TANH, CUT, true>), grid, block, lds, st, p);
    else hipLaunchKernelGGL((k_glr<DT, VEC, TANH, CUT, true>), grid, block, lds, st, p);
    return hipGetLastError();
  }
  const size_t lds = q.nw > 1 ? 2 * maps : 0;
  if (backward) hipLaunchKernelGGL((k_glr_bwd<DT, 1, TANH, CUT, false>), grid, block, lds, st, p);
  else hipLaunchKernelGGL((k_glr<DT, VEC, TANH, CUT, false>), grid, block, lds, st, p);
  return hipGetLastError();
}
template <int DT, int VEC>
hipError_t go_act(const GlrP& p, const Plan& q, bool backward, hipStream_t st) {
  if (p.a.cand_act) return p.a.mask ? go<DT, VEC, true, true>(p, q, backward, st) : go<DT, VEC, true, false>(p, q, backward, st);
  return p.a.mask ? go<DT, VEC, false, true>(p, q, backward, st) : go<DT, VEC, false, false>(p, q, backward, st);
}
template <int DT>
hipError_t go_vec(const GlrP& p, const Plan& q, bool backward, hipStream_t st) {
  return q.vec == 2 ? go_act<DT, 2>(p, q, backward, st) : go_act<DT, 1>(p, q, backward, st);
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
  bool wide = a.D % 2 == 0;
  for (const void* q : f32)
    if (q != a.mask && q != a.lengths && (uintptr_t)q % 8) wide = false;
  wide = wide && aligned(a.gate, a.gate_sb, a.gate_st, es, 2) && aligned(a.cand, a.cand_sb, a.cand_st, es, 2) && aligned(a.out, a.out_sb, a.out_st, es, 2) &&
         aligned(a.dout, a.dout_sb, a.dout_st, es, 2) && aligned(a.dgate, a.dgate_sb, a.dgate_st, es, 2) && aligned(a.dcand, a.dcand_sb, a.dcand_st, es, 2);
  const Plan q = plan_of(a.B, a.T, a.D, wide, backward);
  p.nseg = (int)nseg;
  p.ncb = (int)q.ncb;
  p.ntile = (int)q.ntile;
  if (q.ncb * a.B * (q.chain ? q.ntile : 1) > ops_most_groups(64 * q.nw))
    return ops_fail(HIERTCN_ERR_INVALID, "%lld sequences of %lld channels are too many for one launch: B * ceil(D / 64) is at most 2^26 - 1", (long long)a.B, (long long)a.D);
  if (q.chain) {
    const size_t need = workspace_of(a.B, a.T, a.D);      // (the most that any alignment and direction takes)
    if (!a.workspace || a.workspace_bytes < need || (uintptr_t)a.workspace % 16)
      return ops_fail(HIERTCN_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", need, a.workspace ? a.workspace_bytes : (size_t)0);
    p.map = static_cast<uint64_t*>(a.workspace);
    p.behind = p.map + q.ntile * a.B * a.D;
    p.state0 = reinterpret_cast<float*>(p.map + words_of(q, a.B, a.D));
    p.ticket = reinterpret_cast<unsigned*>(p.state0 + (a.B * a.D + 31) / 32 * 32);
    p.grid = (unsigned)(q.ncb * a.B * q.ntile);
    p.polls = OPS_POLLS;
#ifdef HIERTCN_TEST_HOOKS
    if (const char* polls = getenv("HIERTCN_GLR_TEST_POLLS")) p.polls = (unsigned)atoi(polls);
#endif
  }
  const hipError_t launched = a.dtype == HIERTCN_FP32 ? go_vec<HIERTCN_FP32>(p, q, backward, st) : a.dtype == HIERTCN_BF16 ? go_vec<HIERTCN_BF16>(p, q, backward, st) : go_vec<HIERTCN_FP16>(p, q, backward, st);
  OPS_TRY(launched);
  return HIERTCN_OK;
}

}  // namespace

extern "C" {

size_t hiertcn_glr_record_floats(int64_t B, int64_t T, int64_t D) { return B > 0 && T > 0 && D > 0 ? (size_t)(B * ((T + SEG - 1) / SEG) * D) : 0; }
size_t hiertcn_glr_workspace_bytes(int64_t B, int64_t T, int64_t D) { return B > 0 && T > 0 && D > 0 ? workspace_of(B, T, D) : 0; }
int hiertcn_glr_forward(const hiertcn_glr_t* a, void* stream) { return glr(a, false, reinterpret_cast<hipStream_t>(stream)); }
int hiertcn_glr_backward(const hiertcn_glr_t* a, void* stream) { return glr(a, true, reinterpret_cast<hipStream_t>(stream)); }

}  // extern "C"
