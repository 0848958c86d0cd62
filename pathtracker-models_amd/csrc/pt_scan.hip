// pt_scan.hip — gated linear recurrences over a sequence (include/pt_scan.h).
//
// Mathematics.  A step is h' = a h + b with a, b from the gates of that step
// alone, so n steps together are again h' = P h + q, with P the product of the
// a's and q the result from h = 0.  A chunk of time is cut over the W waves of
// a workgroup, L steps each: every wave reduces its L steps to (P, q), the
// pairs meet in shared memory, each wave composes those before its own and
// walks its L steps from the state it finds -- the sequence is read once.  The
// backward runs the same way from the far end: G_t = (dL/dy_t through y) +
// a_{t+1} G_{t+1}, with the states recomputed in f32 from the one kept at each
// chunk's start.  a is a logistic value, 0 <= a <= 1, so products can only
// underflow, never overflow.
//
// Layout.  A lane owns a column (channel, inner), so every load of a wave is 64
// neighbouring elements of one step.  Two 16-bit columns a lane would halve the
// loads, but what a step keeps until its gradient is known then passes 128
// registers: the backward spilled and took 3.1 times as long.
//
// Where the columns do not fill the card the time axis is also cut over
// workgroups, a chunk each (the chain): a workgroup reduces its chunk to (P, q)
// as above, publishes the pair, takes the pairs of the chunks before its own
// and finishes its chunk from its registers.  The pairs are always joined in
// the same order, so the results do not depend on timing.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "pt_scan.h"

#ifndef PT_SRC_HASH
#define PT_SRC_HASH "unknown"
#endif

namespace {

thread_local char g_err[256] = "";

int fail(int code, const char* msg) {
  snprintf(g_err, sizeof(g_err), "%s", msg);
  return code;
}

// Waves of a workgroup of the chain.  A longer chunk pays the joining less often,
// two workgroups a compute unit hide it better: 32 tiles of 16384 steps, leaky
// bf16, forward 72 us with 8 waves and 64 with 16, backward 93 and 99.
constexpr int CHAIN_FWD = 16, CHAIN_BWD = 8;
constexpr int GROUP = 32;        // chunks after which the chain hands a state on, so that joins stay short
static_assert(GROUP % CHAIN_FWD == 0 && GROUP % CHAIN_BWD == 0 && (GROUP & (GROUP - 1)) == 0,
              "a join is shared out evenly over the waves");
static_assert(CHAIN_FWD == 2 * CHAIN_BWD, "the forward's chunks are two of the backward's, as without the chain");

// One kind of sequence tensor (all gates share their strides): strides in bytes.
struct Strides {
  int64_t b, c, t;
};

struct Args {
  const char* x[4];        // the gates
  char* dx[4];             // their gradients
  char* y;                 // the output, or dy in the backward
  Strides xs, ds, ys;
  const float* h0;
  const int64_t* len;
  float* h_last;
  float* c_last;
  const float* d_h_last;
  const float* d_c_last;
  float* d_h0;
  float* saved;            // [chunk of the backward][B][C N]: the state before it (the first: h0)
  uint32_t* ticket;        // the chain: the next workgroup's number
  uint64_t* pairs;         // the chain: [chunk][B][C N] published pairs (P, q)
  uint64_t* states;        // the chain: [group][B][C N] published pairs (1, state)
  int64_t cols_all;        // B C N
  int64_t C, N;
  int64_t cg, groups;      // channels per column group, groups per batch row
  int64_t outer;           // B groups
  int T;                   // steps
  int tiles, segs;         // column tiles of a row; chunks of the chain
};

template <typename T, int V> using vec = T __attribute__((ext_vector_type(V)));

// A constant in a scalar register: as a literal it would need the short encoding,
// which takes no |x| or -x of its operand, at one more instruction a use.
__device__ __forceinline__ float in_scalar(float c) {
  asm("" : "+s"(c));
  return c;
}

// e^-Nx for x >= 0, N a power of two.  ACC (f32 data): the product x log2(e) is carried in two
// parts, which keeps the error at an ulp for large x too; for 16-bit data the
// single product's error (x 2^-24 relative) is far below the data's step.
template <bool ACC, int N = 1> __device__ __forceinline__ float exp_minus(float x) {
  constexpr float L2E = N * 1.44269502f, L2E_LO = N * 1.92596303e-8f, LN2 = 0.693147182f;
  if constexpr (ACC) {
    x = x > 104.f ? 104.f : x;                 // (inf would make the low part NaN; NaN stays)
    const float c = in_scalar(L2E), t = x * c;
    const float lo = __builtin_fmaf(x, L2E_LO, __builtin_fmaf(x, c, -t));
    const float r = __builtin_amdgcn_exp2f(-t);
    return __builtin_fmaf(r, -lo * LN2, r);
  } else {
    return __builtin_amdgcn_exp2f(x * in_scalar(-L2E));
  }
}

template <bool ACC> __device__ __forceinline__ float recip(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  if constexpr (ACC) return __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r);
  return r;
}

// s(x), s(-x) and their product, each to full relative accuracy (1 - s would
// cancel).  What a caller does not use costs nothing.
struct Logistic { float s, sm, p; };
template <bool ACC> __device__ __forceinline__ Logistic logistic(float x) {
  const float e = exp_minus<ACC>(__builtin_fabsf(x));
  const float big = recip<ACC>(1.f + e), small = e * big;
  return {x >= 0.f ? big : small, x >= 0.f ? small : big, small * big};
}

// 1 - e, e = e^-2x, for x >= 0 and 16-bit data.  Where x is small the difference cancels
// (and is 0 below 2^-25), and x is as often the f32 state as the data: below 1/64 the
// series 2x - 2x^2 + 4/3 x^3, which leaves out 1/3 x^3 of it, at most 21 2^-24; from there
// on the ulp of e is at most 32 2^-24 of the difference.  (Five instructions: lstm
// f16 2 x 2048 x 6400 forward 69 us, 64 without them; the clips below 138 and 138.)
__device__ __forceinline__ float one_minus(float e, float x) {
  const float n = x * __builtin_fmaf(x, __builtin_fmaf(x, 4.f / 3.f, -2.f), 2.f);
  return x < 1.f / 64.f ? n : 1.f - e;
}

// tanh(x) and its derivative 4 e / (1 + e)^2, e = exp(-2|x|).  f32 data: the
// odd series below 0.35 (next term 2e-9 relative), where 1 - e would cancel.
template <bool ACC> __device__ __forceinline__ float tanh_d(float x, float& d) {
  const float ax = __builtin_fabsf(x);
  const float e = exp_minus<ACC, 2>(ax), r = recip<ACC>(1.f + e);
  d = 4.f * e * r * r;
  if constexpr (!ACC) return __builtin_copysignf(one_minus(e, ax) * r, x);
  const float t = __builtin_copysignf((1.f - e) * r, x);
  const float q = x * x;
  float p = -1382.f / 155925.f;
  p = __builtin_fmaf(p, q, 62.f / 2835.f);
  p = __builtin_fmaf(p, q, -17.f / 315.f);
  p = __builtin_fmaf(p, q, 2.f / 15.f);
  p = __builtin_fmaf(p, q, -1.f / 3.f);
  return ax < 0.35f ? __builtin_fmaf(x * q, p, x) : t;
}

// For 16-bit data: what s(x) is the reciprocal of, 1 + e^-x (infinite below -88, where
// s(x) is then 0), and s(x) tanh(v) over one reciprocal.  A fifth fewer instructions a
// step of the lstm's forward than with the functions above (both without the series): 64 clips of 64 frames of
// 25 x 32 x 32 162 to 145 us, 2 x 2048 x 6400 79 to 67.
__device__ __forceinline__ float logistic_denom(float x) {
  return 1.f + __builtin_amdgcn_exp2f(x * in_scalar(-1.44269502f));
}
__device__ __forceinline__ float gated_tanh(float denom, float v) {
  const float av = __builtin_fabsf(v), e = exp_minus<false, 2>(av);
  return __builtin_copysignf(one_minus(e, av), v) * recip<false>(denom * (1.f + e));
}

// Shared memory between the waves of a workgroup: order LDS traffic alone, so
// that the loads in flight for the next chunk are not waited for.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A global address that every lane of the wave holds alike, kept in scalar
// registers: a step's address is then a scalar plus one 32-bit lane offset for
// all steps.  (Left to itself the compiler keeps a 64-bit vector pointer each.)
using gptr = __attribute__((address_space(1))) char*;
__device__ __forceinline__ gptr scalar(const char* p) {
  uint64_t u = (uint64_t)p;
  asm("" : "+s"(u));
  return (gptr)u;
}
// A lane's 32-bit offset, seen by the compiler as one where it is used (hoisted
// out of the loop as a 64-bit value it would no longer fold into the access).
__device__ __forceinline__ uint32_t offset32(uint32_t off) {
  asm("" : "+v"(off));
  return off;
}
// The same for a scalar: what depends on it is computed where it is used (16
// lane masks kept over the loop would be more than the scalar registers hold).
__device__ __forceinline__ int here(int k) {
  asm("" : "+s"(k));
  return k;
}
template <typename T> using gval = __attribute__((address_space(1))) T;

// Where a workgroup works: column tile, row, chunk of the chain; and a lane's column.
struct Where {
  int seg, lane, wave, end;  // `end`: the batch row's
  int64_t b, c0;             // batch row; the group's first channel
  bool on;                   // this lane's column exists
  int64_t state;             // this lane's column in [B][C][N]
  uint32_t off_c, off_n;     // channel in the group, position in the inner axis

  __device__ __forceinline__ Where(const Args& a, uint32_t id) {    // the host keeps the grid below 2^26
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = id % (uint32_t)a.tiles;
    id /= (uint32_t)a.tiles;
    const uint32_t o = id % (uint32_t)a.outer;
    seg = (int)(id / (uint32_t)a.outer);
    const uint32_t br = o / (uint32_t)a.groups;
    b = br;
    c0 = (int64_t)(o - br * (uint32_t)a.groups) * a.cg;
    const uint32_t cols = (uint32_t)(a.cg * a.N);
    uint32_t j = tile * 64 + lane;
    on = j < cols;
    j = on ? j : 0;          // an idle lane reads column 0 and stores nothing
    off_c = a.cg == 1 ? 0 : j / (uint32_t)a.N;
    off_n = j - off_c * (uint32_t)a.N;
    state = (b * a.C + c0) * a.N + j;
    end = a.T;
    if (a.len) {
      const int64_t n = a.len[b];
      end = n < 0 ? 0 : n < a.T ? (int)n : a.T;
    }
  }
  // byte offset of this lane within a step (fits 32 bits: the host checks)
  __device__ __forceinline__ uint32_t lane_off(const Strides& s, int size) const {
    return (uint32_t)(off_c * s.c) + off_n * (uint32_t)size;
  }
  // byte offset of the group at step t
  __device__ __forceinline__ int64_t base(const Strides& s, int t) const {
    return b * s.b + c0 * s.c + (int64_t)t * s.t;
  }
};

// L steps from p on; of which `live` are read, the others 0.
template <typename T, int L>
__device__ __forceinline__ void load_steps(T (&r)[L], const char* p, int64_t st, uint32_t off, int live) {
  if (live >= L) {
    off = offset32(off);
#pragma unroll
    for (int l = 0; l < L; ++l, p += st) r[l] = *(const gval<T>*)(scalar(p) + off);
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l, p += st) {
      T v = (T)0.f;
      if (l < live) v = *(const gval<T>*)(scalar(p) + offset32(off));
      r[l] = v;
    }
  }
}

// The same for stores: steps from `live` on are written as 0, from `room` on not at all.
template <typename T, int L>
__device__ __forceinline__ void store_steps(const T (&r)[L], char* p, int64_t st, uint32_t off, int live, int room) {
  if (live >= L) {
    off = offset32(off);
#pragma unroll
    for (int l = 0; l < L; ++l, p += st) *(gval<T>*)(scalar(p) + off) = r[l];
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l, p += st)
      if (l < room) *(gval<T>*)(scalar(p) + offset32(off)) = l < live ? r[l] : (T)0.f;
  }
}

// Registers whose contents no longer matter (else a loop that loads them in one
// branch copies the old contents in the other).  Written in front of that branch:
// in its else, the stores of both were merged to one of a chosen address, and the
// array lay in scratch memory.
template <typename T, int L> __device__ __forceinline__ void forget(T (&r)[L]) {
#pragma unroll
  for (int l = 0; l < L; ++l) asm("" : "=v"(r[l]));
}

// Values that are to be there at this point: what was loaded for them is free for
// the next loads, and a rare branch that makes them is not turned into selects.
template <int L> __device__ __forceinline__ void settle(float (&r)[L]) {
#pragma unroll
  for (int l = 0; l < L; ++l) asm volatile("" : "+v"(r[l]));
}

// An element as f32 in a register of its own (seen through, |x| of a 16-bit
// element becomes integer arithmetic instead of a modifier of the next operand).
template <typename T> __device__ __forceinline__ float as_f32(T x) {
  float f = (float)x;
  asm("" : "+v"(f));
  return f;
}

template <int FORM> constexpr int gates_of() { return FORM == PT_SCAN_LEAKY ? 2 : 4; }
// Steps of one wave in a chunk of the backward, as many as stay in 128 registers
// beside the next chunk's loads; the forward keeps less per step and takes twice
// as many.  In the chain a chunk is alone and has the registers of two.
template <int FORM> constexpr int back_steps() { return FORM == PT_SCAN_LEAKY ? 8 : 4; }
template <int FORM> constexpr int chain_steps() { return FORM == PT_SCAN_LEAKY ? 16 : 8; }

using f32x2 = vec<float, 2>;

// ------------------------------------------------------------------ a wave's steps, forward

template <int FORM, typename T, int L> struct Fwd {
  static constexpr int G = gates_of<FORM>();
  static constexpr bool LSTM = FORM == PT_SCAN_LSTM, ACC = sizeof(T) == 4;
  float A[L], B[L], O[L];        // a; b, then the states, then y; lstm: s(o), for 16 bits 1 / s(o)

  // From what was loaded.  out_here: some y is made of these steps.
  __device__ __forceinline__ void make(const T (&raw)[G][L], bool out_here) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      if constexpr (!LSTM) {
        const Logistic g = logistic<ACC>(as_f32(raw[0][l]));
        A[l] = g.sm;
        B[l] = g.s * as_f32(raw[1][l]);
      } else if constexpr (ACC) {
        float d;
        A[l] = logistic<ACC>(as_f32(raw[1][l])).s;
        B[l] = logistic<ACC>(as_f32(raw[0][l])).s * tanh_d<ACC>(as_f32(raw[2][l]), d);
      } else {
        A[l] = recip<ACC>(logistic_denom(as_f32(raw[1][l])));
        B[l] = gated_tanh(logistic_denom(as_f32(raw[0][l])), as_f32(raw[2][l]));
      }
      asm volatile("" : "+v"(A[l]), "+v"(B[l]));        // (one after the other, not all at once)
    }
    if constexpr (LSTM) {
      forget(O);
      if (out_here) {
#pragma unroll
        for (int l = 0; l < L; ++l)
          if constexpr (ACC) O[l] = logistic<ACC>(as_f32(raw[3][l])).s;
          else O[l] = logistic_denom(as_f32(raw[3][l]));
      }
    }
    settle(A);
    settle(B);
  }
  // Behind the row's end the state stays.
  __device__ __forceinline__ void end_row(int live) {
    if (live >= L) return;
#pragma unroll
    for (int l = 0; l < L; ++l)
      if (l >= live) { A[l] = 1.f; B[l] = 0.f; }
    settle(A);
    settle(B);
  }
  __device__ __forceinline__ f32x2 piece() const {
    f32x2 e = {A[0], B[0]};
#pragma unroll
    for (int l = 1; l < L; ++l) e = f32x2{e[0] * A[l], __builtin_fmaf(A[l], e[1], B[l])};
    return e;
  }
  // The steps from state c on: y and h_last are written, the state after them returned.
  __device__ __forceinline__ float finish(const Args& a, const Where& w, float c, int t0, int live, int room, bool seq,
                                          bool out_here, char* yp, uint32_t yo) {
#pragma unroll
    for (int l = 0; l < L; ++l) B[l] = c = __builtin_fmaf(A[l], c, B[l]);
    if constexpr (LSTM) {
      if (out_here) {
#pragma unroll
        for (int l = 0; l < L; ++l) {
          float d;
          if constexpr (ACC) B[l] = O[l] * tanh_d<ACC>(B[l], d);
          else B[l] = gated_tanh(O[l], B[l]);
        }
        if (a.h_last && t0 < w.end && w.end - t0 <= L && w.on) {
#pragma unroll
          for (int l = 0; l < L; ++l)
            if (t0 + l == w.end - 1) a.h_last[w.state] = B[l];
        }
      }
    }
    if (seq) {
      T out[L];
#pragma unroll
      for (int l = 0; l < L; ++l) out[l] = (T)B[l];
      if (w.on) store_steps(out, yp, a.ys.t, yo, live, room);
    }
    return c;
  }
};

// The states after a row's last step (lstm: h_last comes with that step's y, and
// is 0 for a row without one).
template <int FORM> __device__ __forceinline__ void last_states(const Args& a, const Where& w, float c) {
  if (!w.on) return;
  if (a.c_last) a.c_last[w.state] = c;
  if (a.h_last && FORM == PT_SCAN_LEAKY) a.h_last[w.state] = c;
  if (a.h_last && FORM == PT_SCAN_LSTM && w.end == 0) a.h_last[w.state] = 0.f;
}

// Forward, a workgroup walking a column tile's whole row, M times the backward's
// steps a wave; each chunk's loads are sent off before the one in front of it is
// finished.  Bound by memory where there are columns enough: leaky f32, 32 clips of 64 frames of 32 x 32 x 32 (805 MB) in
// 159 us, 5.1 TB/s (a copy of 4 GiB reaches 4.8).  For 16 bits the arithmetic is
// nearly as long as the loads: lstm bf16, 64 clips of 64 frames of 25 x 32 x 32
// without y (629 MB), 138 us, 4.6 TB/s, and 172 in turn with its backward; lstm f32,
// 32 of these clips with y (1049 MB), 226 us, 4.6 TB/s.  Of rows of unequal length the longest decides, where a
// compute unit has one: leaky bf16 8 x 2048 x 2048, 68% of the steps live,
// 40 us, 3.9 TB/s.
template <int FORM, typename T, int W, int M>
__global__ __launch_bounds__(64 * W, 4) void k_scan_fwd(Args a) {
  constexpr int G = gates_of<FORM>(), L = M * back_steps<FORM>(), CH = W * L;
  constexpr bool LSTM = FORM == PT_SCAN_LSTM;
  // The waves' (P, q).  Two sets, used in turn: a wave writes a set again only
  // behind a barrier that every wave reaches after its last read of it, so one
  // barrier a chunk does.
  __shared__ f32x2 pq[2][W][64];
  const Where w(a, blockIdx.x);
  const bool seq = a.y != nullptr;
  auto out_in = [&](int t0) { return seq || (LSTM && t0 < w.end && w.end - t0 <= L); };

  float carry = a.h0 ? a.h0[w.state] : 0.f;
  const int mine = w.wave * L;                          // this wave's first step
  const int64_t x_at = w.base(a.xs, mine), x_step = a.xs.t * CH;
  const uint32_t xo = w.lane_off(a.xs, sizeof(T));
  const char* xp[G];
#pragma unroll
  for (int g = 0; g < G; ++g) xp[g] = a.x[g] + x_at;
  char* yp = seq ? a.y + w.base(a.ys, mine) : nullptr;
  const uint32_t yo = seq ? w.lane_off(a.ys, sizeof(T)) : 0;

  T raw[G][L];
  auto fetch = [&](int t0) {
#pragma unroll
    for (int g = 0; g < (LSTM ? 3 : 2); ++g) load_steps(raw[g], xp[g], a.xs.t, xo, w.end - t0);
    if constexpr (LSTM) {                               // o is wanted for y, or at the row's last step
      forget(raw[3]);
      if (out_in(t0)) load_steps(raw[3], xp[3], a.xs.t, xo, w.end - t0);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) xp[g] += x_step;
  };
  fetch(mine);

  int par = 0;
  for (int t = 0; t < a.T; t += CH) {
    const int t0 = t + mine, live = w.end - t0, room = a.T - t0;
    if (t >= w.end) {                                   // the whole chunk is behind the row's end
      if (!seq) break;
      if (w.on) store_steps(raw[0], yp, a.ys.t, yo, 0, room);
      yp += a.ys.t * CH;
      continue;
    }
    Fwd<FORM, T, L> f;
    f.make(raw, out_in(t0));
    if (t + CH < w.end) {
      fetch(t0 + CH);
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g) forget(raw[g]);
    }
    f.end_row(live);

    float cin = carry;
    if constexpr (W > 1) {
      pq[par][w.wave][w.lane] = f.piece();
      lds_barrier();
      // compose: the state before this wave's steps, and the one after the chunk
      const int wave = here(w.wave);
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const f32x2 e = pq[par][k][w.lane];
        cin = k == wave ? carry : cin;
        carry = __builtin_fmaf(e[0], carry, e[1]);
      }
      par ^= 1;
      // where the backward's chunks begin
      if constexpr (M == 2) {
        if (a.saved && (w.wave == 0 || w.wave == W / 2) && t0 > 0 && t0 < a.T && w.on)
          a.saved[(t0 / (CH / 2) - 1) * a.cols_all + w.state] = cin;
      }
    }
    const float after = f.finish(a, w, cin, t0, live, room, seq, out_in(t0), yp, yo);
    if constexpr (W == 1) carry = after;
    if (seq) yp += a.ys.t * CH;
  }
  if (w.wave == 0) last_states<FORM>(a, w, carry);
}

// ------------------------------------------------------------------ a wave's steps, backward

template <int FORM, typename T, int L> struct Bwd {
  static constexpr int G = gates_of<FORM>();
  static constexpr bool LEAKY = FORM == PT_SCAN_LEAKY, ACC = sizeof(T) == 4;
  // a; what the gradients are made of; dy, then dL/dh_t through y_t
  float A[L], K0[L], K1[L], D[L];
  float B[L], K2[L], O[L], OP[L];                       // lstm

  __device__ __forceinline__ void make(const T (&raw)[G][L], const T (&rdy)[L], bool enters) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      D[l] = (float)rdy[l];
      if constexpr (LEAKY) {
        const Logistic z = logistic<ACC>(as_f32(raw[0][l]));
        A[l] = z.sm;
        K1[l] = z.s;
        K0[l] = as_f32(raw[1][l]);
      } else {
        const Logistic f = logistic<ACC>(as_f32(raw[1][l])), i = logistic<ACC>(as_f32(raw[0][l]));
        float d;
        const float th = tanh_d<ACC>(as_f32(raw[2][l]), d);
        A[l] = f.s;
        B[l] = i.s * th;
        K0[l] = i.p * th;
        K1[l] = f.p;
        K2[l] = i.s * d;
      }
    }
    if constexpr (!LEAKY) {
      forget(O);
      forget(OP);
      if (enters) {
#pragma unroll
        for (int l = 0; l < L; ++l) {
          const Logistic g = logistic<ACC>(as_f32(raw[3][l]));
          O[l] = g.s;
          OP[l] = g.p;
        }
      }
      settle(B);
      settle(K2);
    }
    settle(A);
    settle(D);
    settle(K0);
    settle(K1);
  }
  __device__ __forceinline__ void end_row(int live) {   // behind the row's end: h' = h, dx = 0
    if (live >= L) return;
#pragma unroll
    for (int l = 0; l < L; ++l)
      if (l >= live) {
        A[l] = 1.f;
        if constexpr (LEAKY) K1[l] = 0.f; else B[l] = 0.f;
      }
    settle(A);
    if constexpr (LEAKY) settle(K1); else settle(B);
  }
  __device__ __forceinline__ f32x2 piece() const {
    f32x2 e = {A[0], LEAKY ? K1[0] * K0[0] : B[0]};
#pragma unroll
    for (int l = 1; l < L; ++l)
      e = f32x2{e[0] * A[l], __builtin_fmaf(A[l], e[1], LEAKY ? K1[l] * K0[l] : B[l])};
    return e;
  }
  // What leaves the steps towards the past when nothing comes from behind.
  __device__ __forceinline__ float gradient_out() const {
    float g = 0.f;
#pragma unroll
    for (int l = L - 1; l >= 0; --l) g = A[l] * (D[l] + g);
    return g;
  }
  // The states, from c on; the o gate's gradient is written.
  __device__ __forceinline__ void walk(const Args& a, const Where& w, float c, int t0, int live, int room, bool enters,
                                       char* dp3, uint32_t dof) {
    if constexpr (LEAKY) {
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const float n = K0[l], s = K1[l];
        K0[l] = (n - c) * (s * A[l]);
        c = __builtin_fmaf(A[l], c, s * n);
      }
    } else {
      if (enters) {
        if (a.d_h_last && t0 < w.end && w.end - t0 <= L) {
          const float e = a.d_h_last[w.state];
#pragma unroll
          for (int l = 0; l < L; ++l) D[l] += t0 + l == w.end - 1 ? e : 0.f;
          settle(D);
        }
#pragma unroll
        for (int l = 0; l < L; ++l) {
          K1[l] *= c;
          c = __builtin_fmaf(A[l], c, B[l]);
          float d;
          const float th = tanh_d<ACC>(c, d);
          OP[l] *= D[l] * th;
          D[l] *= O[l] * d;
        }
      } else {
#pragma unroll
        for (int l = 0; l < L; ++l) {
          K1[l] *= c;
          c = __builtin_fmaf(A[l], c, B[l]);
          OP[l] = 0.f;
        }
      }
      settle(OP);                        // (16-bit values made in both branches went through scratch memory)
      T out[L];
#pragma unroll
      for (int l = 0; l < L; ++l) out[l] = (T)OP[l];
      if (w.on) store_steps(out, dp3, a.ds.t, dof, live, room);
    }
  }
  // The other gates' gradients, with g coming from behind; returns what leaves.
  __device__ __forceinline__ float finish(const Args& a, const Where& w, float g, int live, int room,
                                          char* const (&dp)[G], uint32_t dof) {
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      D[l] += g;
      g = A[l] * D[l];
    }
    auto give = [&](const float (&k)[L], char* p) {
      T out[L];
#pragma unroll
      for (int l = 0; l < L; ++l) out[l] = (T)(D[l] * k[l]);
      if (w.on) store_steps(out, p, a.ds.t, dof, live, room);
    };
    give(K0, dp[0]);
    give(K1, dp[1]);
    if constexpr (!LEAKY) give(K2, dp[2]);
    return g;
  }
};

// lstm: whether any gradient enters through y among the L steps from t0 (without
// a dy it does at the row's last step alone, and o, tanh(c) matter only there).
__device__ __forceinline__ bool enters_in(const Args& a, const Where& w, int t0, int L) {
  return a.y != nullptr || (a.d_h_last && t0 < w.end && w.end - t0 <= L);
}

// The gradient of the state after a row's last step.
template <int FORM> __device__ __forceinline__ float end_gradient(const Args& a, const Where& w) {
  const float* end = FORM == PT_SCAN_LEAKY ? a.d_h_last : a.d_c_last;
  return end ? end[w.state] : 0.f;
}

// Backward, a workgroup walking a column tile's whole row from its end.  Each
// chunk is walked twice, both times from registers: forward from the kept state,
// then back.  The shapes of the forward: leaky f32 (1342 MB) 261 us, 5.1 TB/s; lstm
// bf16 (1468 MB) 331 us, 4.4 TB/s, and 346 in turn with its forward; lstm f32 with dy
// (1887 MB) 375 us, 5.0 TB/s; leaky bf16 of unequal rows (271 MB) 78 us, 3.5 TB/s.
template <int FORM, typename T, int W>
__global__ __launch_bounds__(64 * W, 4) void k_scan_bwd(Args a) {
  constexpr int G = gates_of<FORM>(), L = back_steps<FORM>(), CH = W * L;
  constexpr bool LEAKY = FORM == PT_SCAN_LEAKY;
  __shared__ f32x2 pq[2][W][64];              // forward (P, q); two sets in turn, as in the forward
  __shared__ float gq[2][W][64];              // backward q (its P is the same)
  const Where w(a, blockIdx.x);
  const bool has_dy = a.y != nullptr;
  float carry = end_gradient<FORM>(a, w);

  // chunks from the last to the first
  int t = (a.T - 1) / CH * CH;
  const int last = t + w.wave * L;                      // this wave's first step in the last chunk
  const int64_t x_at = w.base(a.xs, last), x_step = a.xs.t * CH;
  const uint32_t xo = w.lane_off(a.xs, sizeof(T));
  const int64_t d_at = w.base(a.ds, last), d_step = a.ds.t * CH;
  const uint32_t dof = w.lane_off(a.ds, sizeof(T));
  const char* xp[G];
  char* dp[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    xp[g] = a.x[g] + x_at;
    dp[g] = a.dx[g] + d_at;
  }
  const char* yp = has_dy ? a.y + w.base(a.ys, last) : nullptr;
  const uint32_t yo = has_dy ? w.lane_off(a.ys, sizeof(T)) : 0;

  T raw[G][L], rdy[L];
  float nst = 0.f;                                      // the state before the fetched chunk
  auto fetch = [&](int tc) {
    const int t0 = tc + w.wave * L, live = w.end - t0;
#pragma unroll
    for (int g = 0; g < (LEAKY ? 2 : 3); ++g) load_steps(raw[g], xp[g], a.xs.t, xo, live);
    if constexpr (!LEAKY) {
      forget(raw[3]);
      if (enters_in(a, w, t0, L)) load_steps(raw[3], xp[3], a.xs.t, xo, live);
    }
    if (has_dy) load_steps(rdy, yp, a.ys.t, yo, live);
    const float* s = tc > 0 ? a.saved + (tc / CH - 1) * a.cols_all : a.h0;
    nst = s ? s[w.state] : 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) xp[g] -= x_step;
    if (has_dy) yp -= a.ys.t * CH;
  };
#pragma unroll
  for (int l = 0; l < L; ++l) rdy[l] = (T)0.f;

  for (; t >= 0 && t >= w.end; t -= CH) {               // behind the row's end dx is only cleared
#pragma unroll
    for (int g = 0; g < G; ++g) {
      xp[g] -= x_step;
      if (w.on) store_steps(rdy, dp[g], a.ds.t, dof, 0, a.T - (t + w.wave * L));
      dp[g] -= d_step;
    }
    if (has_dy) yp -= a.ys.t * CH;
  }
  if (t >= 0) fetch(t);
  int par = 0;
  for (; t >= 0; t -= CH) {
    const int t0 = t + w.wave * L, live = w.end - t0, room = a.T - t0;
    const bool enters = enters_in(a, w, t0, L);
    float cin = nst;
    Bwd<FORM, T, L> b;
    b.make(raw, rdy, enters);
    if (t > 0) {
      fetch(t - CH);
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g) forget(raw[g]);
      if (has_dy) forget(rdy);
    }
    b.end_row(live);

    float gin = carry;
    if constexpr (W > 1) {
      pq[par][w.wave][w.lane] = b.piece();
      if constexpr (LEAKY) gq[par][w.wave][w.lane] = b.gradient_out();      // y = h: dy needs no state
      lds_barrier();
      const int wave = here(w.wave);
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        const f32x2 e = pq[par][k][w.lane];
        cin = k < wave ? __builtin_fmaf(e[0], cin, e[1]) : cin;
      }
    }
    b.walk(a, w, cin, t0, live, room, enters, dp[G - 1], dof);
    if constexpr (W > 1) {
      if constexpr (!LEAKY) {
        gq[par][w.wave][w.lane] = b.gradient_out();
        lds_barrier();
      }
      const int wave = here(w.wave);
#pragma unroll
      for (int k = W - 1; k >= 0; --k) {
        gin = k == wave ? carry : gin;
        carry = __builtin_fmaf(pq[par][k][w.lane][0], carry, gq[par][k][w.lane]);
      }
      par ^= 1;
    }
    const float out = b.finish(a, w, gin, live, room, dp, dof);
    if constexpr (W == 1) carry = out;
#pragma unroll
    for (int g = 0; g < G; ++g) dp[g] -= d_step;
  }
  if (w.wave == 0 && w.on && a.d_h0) a.d_h0[w.state] = carry;
}

// ------------------------------------------------------------------ the chain
//
// Workgroups take numbers from a ticket, so whatever a workgroup waits for was
// taken up before it and waits itself only for still earlier ones: every wait
// ends, whatever order the card starts them in.  Every chunk publishes what a
// later one could wait for, also behind its row's end, so that the waits do not
// hang on what `lengths` holds either.  A pair is one 64-bit word that
// is written once, so a reader sees none of it or all of it, and needs no fence:
// nothing but the word is handed over.  NOT_YET is what no pair can be (its P
// would be a NaN of a form that is never published).
//
// A chunk is loaded, joined and stored by one workgroup that does nothing else:
// leaky bf16, 16384 steps of 2048 columns (201 MB), 57 us, 3.5 TB/s; lstm bf16, 2 rows
// of 8192 steps of 512 (84 and 151 MB), forward 31 us and backward 55 us, 2.7 TB/s
// both; the same in f32 51 and 73 us, 3.3 and 4.1 TB/s.  Twice the bytes do not take
// twice the time: part of it is a chunk's own, whatever it holds.  Waves wait 58 to 63 %
// of their cycles and issue vector instructions in about a tenth; the counters do not
// tell the wait for a join from that for loads.  Reading the
// sequence twice instead (every chunk's pair, then the walk) took, at 16384 steps
// of 2048 columns, for leaky f32 128 us and in the backward 194, against 95 and
// 132 here; for lstm bf16 128 and 248, against 113 and 193.  A workgroup that
// sends off its next chunk's loads before it joins is slower (leaky bf16 92 us):
// loads return in order, so the join then waits for the next chunk too.

constexpr uint64_t NOT_YET = ~(uint64_t)0;
constexpr int CHAIN_HEAD = 256;          // bytes of the ticket, in front of the pairs

// The ticket to 0 and every pair to NOT_YET, `n` times 16 bytes (2 to 4 us; a kernel,
// as a memory operation recorded into a graph is not safe to replay here).
__global__ __launch_bounds__(256) void k_chain_clear(vec<uint32_t, 4>* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    p[i] = i < CHAIN_HEAD / 16 ? (vec<uint32_t, 4>)(0u) : (vec<uint32_t, 4>)(~0u);
}

__device__ __forceinline__ uint32_t chain_number(uint32_t* ticket) {
  __shared__ uint32_t id;
  if (threadIdx.x == 0) id = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(id);
}

__device__ __forceinline__ void publish(uint64_t* slot, float p, float q) {
  const uint32_t pb = p != p ? 0x7fc00000u : __builtin_bit_cast(uint32_t, p);
  __hip_atomic_store(slot, (uint64_t)__builtin_bit_cast(uint32_t, q) << 32 | pb, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t* slot) {
  return __hip_atomic_load(slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A chunk behind its row's end: nobody uses its pair, nor the state after it.
__device__ __forceinline__ void publish_idle(const Args& a, const Where& w, bool chunk, bool group) {
  if (w.wave != 0 || !w.on) return;
  if (chunk) publish(a.pairs + w.seg * a.cols_all + w.state, 1.f, 0.f);
  if (group) publish(a.states + w.seg / GROUP * a.cols_all + w.state, 1.f, 0.f);
}
// The pair, from a first look at it.  (Idle lanes look at column 0's, which is published as well.)
__device__ __forceinline__ f32x2 await(const uint64_t* slot, uint64_t v) {
  while (__any(v == NOT_YET)) {
    __builtin_amdgcn_s_sleep(1);
    v = peek(slot);
  }
  return f32x2{__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32))};
}

// One wave's part of the pairs of `count` chunks from `slot` on, `step` words apart,
// joined in this order: the waves look at them side by side, one round trip to
// memory for all.
template <int W>
__device__ __forceinline__ f32x2 join(const uint64_t* slot, int64_t step, int count, int wave) {
  constexpr int N = GROUP / W;
  count -= wave * N;
  slot += wave * N * step;
  uint64_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < count ? peek(slot + i * step) : 0;
  f32x2 e = {1.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < count) {
      const f32x2 n = await(slot + i * step, v[i]);
      e = f32x2{e[0] * n[0], __builtin_fmaf(n[0], e[1], n[1])};
    }
  return e;
}

// Forward: reduce, publish, join what lies before, walk.
template <int FORM, typename T> __global__ __launch_bounds__(64 * CHAIN_FWD, 4) void k_chain_fwd(Args a) {
  constexpr int W = CHAIN_FWD, G = gates_of<FORM>(), L = chain_steps<FORM>(), CH = W * L;
  constexpr bool LSTM = FORM == PT_SCAN_LSTM;
  __shared__ f32x2 pq[W][64], pj[W][64];  // the waves' pieces; their parts of the join
  __shared__ float cs[64];               // what the join starts from
  const Where w(a, chain_number(a.ticket));
  const int t_beg = w.seg * CH, t0 = t_beg + w.wave * L, live = w.end - t0, room = a.T - t0;
  const bool seq = a.y != nullptr;
  char* yp = seq ? a.y + w.base(a.ys, t0) : nullptr;
  const uint32_t yo = seq ? w.lane_off(a.ys, sizeof(T)) : 0;
  const bool more = w.seg + 1 < a.segs, hands_on = more && (w.seg + 1) % GROUP == 0;
  if (t_beg >= w.end) {                  // behind the row's end
    publish_idle(a, w, more, hands_on);
    const T none[L] = {};
    if (seq && w.on) store_steps(none, yp, a.ys.t, yo, 0, room);
    if (w.seg == 0 && w.wave == 0) last_states<FORM>(a, w, a.h0 ? a.h0[w.state] : 0.f);
    return;
  }
  const bool out_here = seq || (LSTM && t0 < w.end && w.end - t0 <= L);
  const int64_t x_at = w.base(a.xs, t0);
  const uint32_t xo = w.lane_off(a.xs, sizeof(T));
  T raw[G][L];
#pragma unroll
  for (int g = 0; g < (LSTM ? 3 : 2); ++g) load_steps(raw[g], a.x[g] + x_at, a.xs.t, xo, live);
  if constexpr (LSTM) {
    forget(raw[3]);
    if (out_here) load_steps(raw[3], a.x[3] + x_at, a.xs.t, xo, live);
  }
  Fwd<FORM, T, L> f;
  f.make(raw, out_here);
  f.end_row(live);
  pq[w.wave][w.lane] = f.piece();
  lds_barrier();
  const int first = w.seg & -GROUP, group = w.seg / GROUP;
  f32x2 own = {1.f, 0.f};                               // wave 0: the chunk's pair
  if (w.wave == 0) {
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const f32x2 n = pq[k][w.lane];
      own = f32x2{own[0] * n[0], __builtin_fmaf(n[0], own[1], n[1])};
    }
    if (more && w.on) publish(a.pairs + w.seg * a.cols_all + w.state, own[0], own[1]);
    if (first == 0) {
      cs[w.lane] = a.h0 ? a.h0[w.state] : 0.f;
    } else {
      const uint64_t* s = a.states + (group - 1) * a.cols_all + w.state;
      cs[w.lane] = await(s, peek(s))[1];
    }
  }
  pj[w.wave][w.lane] = join<W>(a.pairs + first * a.cols_all + w.state, a.cols_all, w.seg - first, w.wave);
  lds_barrier();
  float c = cs[w.lane];
#pragma unroll
  for (int k = 0; k < W; ++k) {
    const f32x2 e = pj[k][w.lane];
    c = __builtin_fmaf(e[0], c, e[1]);
  }
  if (w.wave == 0) {
    const float after = __builtin_fmaf(own[0], c, own[1]);
    if (hands_on && w.on) publish(a.states + group * a.cols_all + w.state, 1.f, after);
    if (t_beg + CH >= w.end) last_states<FORM>(a, w, after);
  }
  for (int k = 0; k < w.wave; ++k) {
    const f32x2 e = pq[k][w.lane];
    c = __builtin_fmaf(e[0], c, e[1]);
  }
  // where the backward's chunks begin
  if (a.saved && (w.wave == 0 || w.wave == W / 2) && t0 > 0 && t0 < a.T && w.on)
    a.saved[(t0 / (CH / 2) - 1) * a.cols_all + w.state] = c;
  f.finish(a, w, c, t0, live, room, seq, out_here, yp, yo);
}

// Backward: the states from the one kept at the chunk's start, then as the forward
// from the far end.
template <int FORM, typename T> __global__ __launch_bounds__(64 * CHAIN_BWD, 4) void k_chain_bwd(Args a) {
  constexpr int W = CHAIN_BWD, G = gates_of<FORM>(), L = chain_steps<FORM>(), CH = W * L;
  constexpr bool LEAKY = FORM == PT_SCAN_LEAKY;
  __shared__ f32x2 pq[W][64], pj[W][64];  // as in the forward; gq: the pieces' q backward
  __shared__ float gq[W][64], cs[64];
  Where w(a, chain_number(a.ticket));
  w.seg = a.segs - 1 - w.seg;            // from the far end
  const int t_beg = w.seg * CH, t0 = t_beg + w.wave * L, live = w.end - t0, room = a.T - t0;
  const bool has_dy = a.y != nullptr;
  const int64_t d_at = w.base(a.ds, t0);
  const uint32_t dof = w.lane_off(a.ds, sizeof(T));
  char* dp[G];
#pragma unroll
  for (int g = 0; g < G; ++g) dp[g] = a.dx[g] + d_at;
  if (t_beg >= w.end) {                  // behind the row's end
    publish_idle(a, w, w.seg > 0, w.seg > 0 && w.seg % GROUP == 0);
    const T none[L] = {};
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (w.on) store_steps(none, dp[g], a.ds.t, dof, 0, room);
    if (w.seg == 0 && w.wave == 0 && w.on && a.d_h0) a.d_h0[w.state] = end_gradient<FORM>(a, w);
    return;
  }
  const bool enters = enters_in(a, w, t0, L);
  const int64_t x_at = w.base(a.xs, t0);
  const uint32_t xo = w.lane_off(a.xs, sizeof(T));
  T raw[G][L], rdy[L] = {};
#pragma unroll
  for (int g = 0; g < (LEAKY ? 2 : 3); ++g) load_steps(raw[g], a.x[g] + x_at, a.xs.t, xo, live);
  if constexpr (!LEAKY) {
    forget(raw[3]);
    if (enters) load_steps(raw[3], a.x[3] + x_at, a.xs.t, xo, live);
  }
  if (has_dy) load_steps(rdy, a.y + w.base(a.ys, t0), a.ys.t, w.lane_off(a.ys, sizeof(T)), live);
  const float* s = w.seg > 0 ? a.saved + (w.seg - 1) * a.cols_all : a.h0;
  float cin = s ? s[w.state] : 0.f;
  Bwd<FORM, T, L> b;
  b.make(raw, rdy, enters);
  b.end_row(live);
  pq[w.wave][w.lane] = b.piece();
  if constexpr (LEAKY) gq[w.wave][w.lane] = b.gradient_out();
  lds_barrier();
  for (int k = 0; k < w.wave; ++k) {
    const f32x2 e = pq[k][w.lane];
    cin = __builtin_fmaf(e[0], cin, e[1]);
  }
  b.walk(a, w, cin, t0, live, room, enters, dp[G - 1], dof);
  if constexpr (!LEAKY) {
    gq[w.wave][w.lane] = b.gradient_out();
    lds_barrier();
  }
  const int far = (w.end - 1) / CH;                     // the row's last chunk
  const int group = w.seg / GROUP, next = (group + 1) * GROUP;
  const int from = next > far ? far : next - 1;         // the last chunk whose pair is joined
  f32x2 own = {1.f, 0.f};                               // wave 0: the chunk's pair
  if (w.wave == 0) {
#pragma unroll
    for (int k = W - 1; k >= 0; --k) {
      const float p = pq[k][w.lane][0];
      own = f32x2{own[0] * p, __builtin_fmaf(p, own[1], gq[k][w.lane])};
    }
    if (w.seg > 0 && w.on) publish(a.pairs + w.seg * a.cols_all + w.state, own[0], own[1]);
    if (next > far) {
      cs[w.lane] = end_gradient<FORM>(a, w);
    } else {
      const uint64_t* st = a.states + (group + 1) * a.cols_all + w.state;
      cs[w.lane] = await(st, peek(st))[1];
    }
  }
  pj[w.wave][w.lane] = join<W>(a.pairs + from * a.cols_all + w.state, -a.cols_all, from - w.seg, w.wave);
  lds_barrier();
  float g = cs[w.lane];
#pragma unroll
  for (int k = 0; k < W; ++k) {
    const f32x2 e = pj[k][w.lane];
    g = __builtin_fmaf(e[0], g, e[1]);
  }
  if (w.wave == 0) {
    const float out = __builtin_fmaf(own[0], g, own[1]);
    if (w.seg > 0 && w.seg % GROUP == 0 && w.on) publish(a.states + group * a.cols_all + w.state, 1.f, out);
    if (w.seg == 0 && w.on && a.d_h0) a.d_h0[w.state] = out;
  }
  for (int k = W - 1; k > w.wave; --k) g = __builtin_fmaf(pq[k][w.lane][0], g, gq[k][w.lane]);
  b.finish(a, w, g, live, room, dp, dof);
}

// One step: element-wise, 16 bytes of the gates a lane where alignment allows.  Bound
// by memory (lstm f32, 64 x 25600, 45.9 MB: 10.2 us, 4.5 TB/s) and by the launch for
// one token (leaky bf16, 1 x 2048: 2.4 us on the device, 5.0 us a call).
template <int FORM, typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(Args a, char* state, Strides ss) {
  constexpr int G = gates_of<FORM>();
  constexpr bool ACC = sizeof(T) == 4;
  const int64_t cols = a.C * a.N;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= a.cols_all) return;
  const int64_t b = i / cols, j = i - b * cols;
  const int64_t c = a.C == 1 ? 0 : j / a.N, n = j - c * a.N;
  auto at = [&](const Strides& s, int size) { return b * s.b + c * s.c + n * size; };
  vec<T, V> x[G], out;
#pragma unroll
  for (int g = 0; g < G; ++g) x[g] = *(const vec<T, V>*)(a.x[g] + at(a.xs, sizeof(T)));
  char* sp = state + at(ss, 4);
  vec<float, V> h = *(const vec<float, V>*)sp;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Logistic g = logistic<ACC>((float)x[0][v]);
    if constexpr (FORM == PT_SCAN_LEAKY) {
      h[v] = __builtin_fmaf(g.sm, h[v], g.s * (float)x[1][v]);
      out[v] = (T)h[v];
    } else {
      float d;
      h[v] = __builtin_fmaf(logistic<ACC>((float)x[1][v]).s, h[v], g.s * tanh_d<ACC>((float)x[2][v], d));
      out[v] = (T)(logistic<ACC>((float)x[3][v]).s * tanh_d<ACC>(h[v], d));
    }
  }
  *(vec<float, V>*)sp = h;
  *(vec<T, V>*)(a.y + at(a.ys, sizeof(T))) = out;
}

// ------------------------------------------------------------------ host

int elem_size(int dtype) { return dtype == PT_SCAN_F32 ? 4 : 2; }
int gates(int form) { return form == PT_SCAN_LEAKY ? 2 : 4; }

int check(const pt_scan_desc* d) {
  if (!d) return fail(PT_SCAN_ERR_ARG, "null scan descriptor");
  if (d->form != PT_SCAN_LEAKY && d->form != PT_SCAN_LSTM) return fail(PT_SCAN_ERR_ARG, "scan: unknown form");
  if (d->dtype < PT_SCAN_F32 || d->dtype > PT_SCAN_F16) return fail(PT_SCAN_ERR_ARG, "scan: unknown dtype");
  if (d->batch < 1 || d->channels < 1 || d->steps < 1 || d->inner < 1)
    return fail(PT_SCAN_ERR_ARG, "scan: batch, channels, steps and inner must be >= 1");
  if (d->steps > (int64_t)1 << 30) return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: steps must be at most 2^30");
  const int64_t big = (int64_t)1 << 40;
  if (d->batch > big || d->channels > big || d->inner > big ||
      (double)d->batch * (double)d->channels * (double)d->inner * (double)d->steps > 1e15)
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: more elements than any device holds");
  if (d->inner >= ((int64_t)1 << 29))
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: inner must be below 2^29");
  return 0;
}

// How a shape is cut; from the descriptor alone, so that forward, backward and
// the size queries agree.
struct Plan {
  int W;                     // 0: the chain
  int64_t chunk, nchunks;    // of the backward; the forward's are two of them
};

// The waves that share a column tile, by the column tiles there are.  The card
// holds 256 workgroups of 16 waves at a time, or 512 of 8 (registers), or 1024
// and more of 4:
//   tiles > 512   4 waves.  More waves only make each chunk's exchange longer
//                 (2048 tiles of 300 steps, leaky bf16: forward 48 us, 58 with 8;
//                 700 of 4096: 262, 269).
//   257 .. 512    8 waves (300 tiles of 4096 steps: 146 us, 162 with 4 or 16).
//   129 .. 256    16 waves: one workgroup a compute unit (180 tiles: 81 us, 136
//                 with 4, 108 with 8).
//   up to 128     the chain, from more than one of its forward's chunks on; else 8
//                 waves.  (4096 steps of leaky bf16, forward and backward: 64
//                 tiles 42 and 47 us, 66 and 107 with 16 waves; 128 tiles 66 and
//                 93, 67 and 136; 256 tiles 127 and 176, 95 and 147.)
// The limits were found with leaky bf16.  The other kinds at 2048 steps, forward /
// backward in us (what the rule takes stands first):
//            leaky f32                    lstm bf16                     lstm f32
//   128  chain 42/72, 16: 37/89      chain 50/106, 16: 68/156     chain 99/126, 16: 110/174
//   180  16: 54/101, chain 62/98     16: 68/159, chain 67/147     16: 121/190, chain 136/175
//   256  16: 82/136, 8: 79/129       16: 80/169, 8: 82/172        16: 146/243, 8: 144/229
//   300  8: 120/199, chain 103/153   8: 127/256, chain 113/239    8: 232/383, chain 215/280
//   512  8: 166/275, 4: 166/266      8: 148/276, 4: 159/337       8: 287/510, 4: 288/471
//   700  4: 235/387, 8: 231/380      4: 214/428, 8: 207/378       4: 421/729, 8: 414/719
// Just above 256 tiles the chain is 7 to 27 % faster for them, at 700 8 waves for lstm
// bf16's backward by 12 %.
// Up to 4 L steps fit a chunk of 4 waves, up to L steps one wave.
Plan plan_of(const pt_scan_desc* d) {
  Plan p;
  const bool leaky = d->form == PT_SCAN_LEAKY;
  const int L = leaky ? back_steps<PT_SCAN_LEAKY>() : back_steps<PT_SCAN_LSTM>();
  const int chain = CHAIN_BWD * (leaky ? chain_steps<PT_SCAN_LEAKY>() : chain_steps<PT_SCAN_LSTM>());
  const int64_t tiles = d->batch * ((d->channels * d->inner + 63) / 64);
  if (d->steps <= L) p.W = 1;
  else if (d->steps <= 4 * L || tiles > 512) p.W = 4;
  else if (tiles > 256) p.W = 8;
  else if (tiles > 128) p.W = 16;
  else p.W = d->steps > 2 * chain ? 0 : 8;
  p.chunk = p.W ? (int64_t)p.W * L : chain;
  p.nchunks = (d->steps + p.chunk - 1) / p.chunk;
  return p;
}

// The chain's scratch for `segs` chunks: the ticket, a pair per chunk, a state per
// group of chunks.
size_t chain_bytes(const pt_scan_desc* d, int64_t segs) {
  const int64_t words = (segs + (segs + GROUP - 1) / GROUP) * d->batch * d->channels * d->inner;
  return CHAIN_HEAD + ((size_t)words * sizeof(uint64_t) + 15) / 16 * 16;
}

// Strides of axes of one element never count: 0, so that they cannot spoil the alignment.
pt_scan_view tidy(const pt_scan_desc* d, const pt_scan_view& v) {
  return pt_scan_view{v.data, d->batch == 1 ? 0 : v.sb, d->channels == 1 ? 0 : v.sc, d->steps == 1 ? 0 : v.st};
}
Strides bytes_of(const pt_scan_view& v, int size) { return Strides{v.sb * size, v.sc * size, v.st * size}; }

// Both halves of the alignment rule: V elements of a lane are one load only if
// every stride and the base keep them aligned and V divides the inner axis.
bool aligned(const pt_scan_view& v, int V, int size) {
  return ((uintptr_t)v.data % (V * size)) == 0 && v.sb % V == 0 && v.sc % V == 0 && v.st % V == 0;
}

bool spans32(const pt_scan_desc* d, const pt_scan_view& v, int size) {
  const double s = ((double)(d->channels - 1) * (double)(v.sc < 0 ? -v.sc : v.sc) + (double)d->inner) * size;
  return v.sc >= 0 && s < 2147483648.0;
}

// The forward takes the backward's short chunk where that holds the whole row: of
// twice the steps a wave, half the waves would have none (lstm bf16 64 x 16 x 4096:
// 20 us, 13 with the short one; leaky f32 2 x 37 x 200: 5.8, 4.8).  Longer rows want
// the long one (leaky bf16 4096 x 16384: 95 us, 107 with the short one).
template <int FORM, typename T, int W>
void launch_rows(const Plan& p, const Args& a, int64_t blocks, bool bwd, hipStream_t s) {
  const dim3 grid((unsigned)blocks), block(64 * W);
  if (bwd) hipLaunchKernelGGL((k_scan_bwd<FORM, T, W>), grid, block, 0, s, a);
  else if (p.nchunks == 1) hipLaunchKernelGGL((k_scan_fwd<FORM, T, W, 1>), grid, block, 0, s, a);
  else if constexpr (W > 1) hipLaunchKernelGGL((k_scan_fwd<FORM, T, W, 2>), grid, block, 0, s, a);
}

template <int FORM, typename T> void launch_chain(const Args& a, int64_t blocks, bool bwd, hipStream_t s) {
  if (bwd) hipLaunchKernelGGL((k_chain_bwd<FORM, T>), dim3((unsigned)blocks), dim3(64 * CHAIN_BWD), 0, s, a);
  else hipLaunchKernelGGL((k_chain_fwd<FORM, T>), dim3((unsigned)blocks), dim3(64 * CHAIN_FWD), 0, s, a);
}

template <int FORM, typename T>
int launch_w(const Plan& p, const Args& a, int64_t blocks, bool bwd, hipStream_t s) {
  switch (p.W) {
    case 0: launch_chain<FORM, T>(a, blocks, bwd, s); break;
    case 1: launch_rows<FORM, T, 1>(p, a, blocks, bwd, s); break;
    case 4: launch_rows<FORM, T, 4>(p, a, blocks, bwd, s); break;
    case 8: launch_rows<FORM, T, 8>(p, a, blocks, bwd, s); break;
    default: launch_rows<FORM, T, 16>(p, a, blocks, bwd, s);
  }
  return hipGetLastError() == hipSuccess ? 0 : fail(PT_SCAN_ERR_HIP, "scan: launch failed");
}

template <int FORM>
int launch_t(int dtype, const Plan& p, const Args& a, int64_t blocks, bool bwd, hipStream_t s) {
  if (dtype == PT_SCAN_F32) return launch_w<FORM, float>(p, a, blocks, bwd, s);
  if (dtype == PT_SCAN_BF16) return launch_w<FORM, __bf16>(p, a, blocks, bwd, s);
  return launch_w<FORM, _Float16>(p, a, blocks, bwd, s);
}

// A launch counts its threads in 32 bits.
bool fits_launch(double blocks, int threads) { return blocks * threads < 4294967296.0; }

// The tensors of a call, checked.
struct Tensors {
  const pt_scan_desc* d;
  int size;
  bool wide;                 // 16 bytes of neighbours lie together and aligned in every one
  bool grouped = true;       // 32-bit offsets reach over the channels of a step
  int rc = 0;

  explicit Tensors(const pt_scan_desc* desc) : d(desc), size(elem_size(desc->dtype)) {
    wide = d->inner % (16 / size) == 0;
  }
  // `count` views of one kind: their pointers and shared strides
  template <typename P> void take(const pt_scan_view* v, int count, P** ptr, Strides& s, int elem) {
    if (rc) return;
    for (int g = 0; g < count; ++g) {
      const pt_scan_view t = tidy(d, v[g]), first = tidy(d, v[0]);
      if (!t.data) { rc = fail(PT_SCAN_ERR_ARG, "scan: null pointer"); return; }
      if ((uintptr_t)t.data % elem) { rc = fail(PT_SCAN_ERR_ARG, "scan: a tensor is not aligned to its elements"); return; }
      if (t.sb != first.sb || t.sc != first.sc || t.st != first.st) {
        rc = fail(PT_SCAN_ERR_UNSUPPORTED, "scan: the gates must share their strides");
        return;
      }
      wide = wide && aligned(t, 16 / size, elem);
      grouped = grouped && spans32(d, t, elem);
      ptr[g] = (P*)t.data;
      s = bytes_of(t, elem);
    }
  }
};

int run(const pt_scan_desc* d, const Plan& p, const Tensors& ts, Args& a, void* workspace, bool bwd, hipStream_t s) {
  // Columns of one channel at a time where the inner axis fills whole tiles, or
  // where the channels of a step reach over more than a 32-bit offset.
  const bool grouped = ts.grouped && d->inner % 64 != 0 &&
                       (double)d->channels * (double)d->inner < 2147483648.0;
  a.C = d->channels;
  a.N = d->inner;
  a.T = (int)d->steps;
  a.cols_all = d->batch * d->channels * d->inner;
  a.cg = grouped ? d->channels : 1;
  a.groups = d->channels / a.cg;
  a.outer = d->batch * a.groups;
  a.segs = p.W ? 1 : (int)(bwd ? p.nchunks : (p.nchunks + 1) / 2);
  const int64_t tiles = (a.cg * a.N + 63) / 64;
  a.tiles = (int)tiles;
  const int threads = 64 * (p.W ? p.W : bwd ? CHAIN_BWD : CHAIN_FWD);
  if (!fits_launch((double)tiles * (double)a.outer * (double)a.segs, threads))
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: more columns and steps than one launch takes");
  if (!p.W) {
    if (!workspace || (uintptr_t)workspace % 16)
      return fail(PT_SCAN_ERR_ARG, "scan: this shape needs a workspace, aligned to 16 bytes");
    a.ticket = (uint32_t*)workspace;
    a.pairs = (uint64_t*)((char*)workspace + CHAIN_HEAD);
    a.states = a.pairs + a.segs * a.cols_all;
    const int64_t n = (int64_t)(chain_bytes(d, a.segs) / 16);
    hipLaunchKernelGGL(k_chain_clear, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 2048)), dim3(256), 0, s,
                       (vec<uint32_t, 4>*)workspace, n);
  }
  const int64_t blocks = tiles * a.outer * a.segs;
  return d->form == PT_SCAN_LEAKY ? launch_t<PT_SCAN_LEAKY>(d->dtype, p, a, blocks, bwd, s)
                                  : launch_t<PT_SCAN_LSTM>(d->dtype, p, a, blocks, bwd, s);
}

}  // namespace

extern "C" {

const char* pt_scan_last_error(void) { return g_err; }
const char* pt_scan_version(void) { return "pt_scan 0.1 gfx950 src " PT_SRC_HASH; }

size_t pt_scan_saved_bytes(const pt_scan_desc* d) {
  if (check(d)) return 0;
  const Plan p = plan_of(d);
  return (size_t)((p.nchunks - 1) * d->batch * d->channels * d->inner) * sizeof(float);
}

size_t pt_scan_workspace_bytes(const pt_scan_desc* d) {
  if (check(d)) return 0;
  const Plan p = plan_of(d);
  return p.W ? 0 : chain_bytes(d, p.nchunks);          // the backward's chunks: the most
}

int pt_scan_forward(const pt_scan_desc* d, const pt_scan_view* x, const float* h0, const int64_t* lengths,
                    const pt_scan_view* y, float* h_last, float* c_last, void* saved, void* workspace,
                    pt_scan_stream_t stream) {
  if (int rc = check(d)) return rc;
  if (!x) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
  const Plan p = plan_of(d);
  Args a{};
  Tensors ts(d);
  ts.take(x, gates(d->form), a.x, a.xs, ts.size);
  if (y && y->data) ts.take(y, 1, &a.y, a.ys, ts.size);
  if (ts.rc) return ts.rc;
  a.h0 = h0; a.len = lengths; a.h_last = h_last; a.c_last = c_last;
  a.saved = p.nchunks > 1 ? (float*)saved : nullptr;
  return run(d, p, ts, a, workspace, false, (hipStream_t)stream);
}

int pt_scan_backward(const pt_scan_desc* d, const pt_scan_view* x, const float* h0, const int64_t* lengths,
                     const pt_scan_view* dy, const float* d_h_last, const float* d_c_last, const void* saved,
                     const pt_scan_view* dx, float* d_h0, void* workspace, pt_scan_stream_t stream) {
  if (int rc = check(d)) return rc;
  if (!x || !dx) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
  const Plan p = plan_of(d);
  Args a{};
  Tensors ts(d);
  ts.take(x, gates(d->form), a.x, a.xs, ts.size);
  ts.take(dx, gates(d->form), a.dx, a.ds, ts.size);
  if (dy && dy->data) ts.take(dy, 1, &a.y, a.ys, ts.size);
  if (ts.rc) return ts.rc;
  if (p.nchunks > 1 && !saved) return fail(PT_SCAN_ERR_ARG, "scan: the backward needs the forward's saved states");
  a.h0 = h0; a.len = lengths; a.d_h_last = d_h_last; a.d_c_last = d_c_last; a.d_h0 = d_h0;
  a.saved = (float*)saved;
  return run(d, p, ts, a, workspace, true, (hipStream_t)stream);
}

int pt_scan_step(const pt_scan_desc* d, const pt_scan_view* x, const pt_scan_view* state, const pt_scan_view* y,
                 pt_scan_stream_t stream) {
  if (int rc = check(d)) return rc;
  if (!x || !state || !y) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
  if (d->steps != 1) return fail(PT_SCAN_ERR_ARG, "scan: a step has steps = 1");
  Args a{};
  Tensors ts(d);
  char* sp = nullptr;
  Strides ss{};
  ts.take(x, gates(d->form), a.x, a.xs, ts.size);
  ts.take(y, 1, &a.y, a.ys, ts.size);
  ts.take(state, 1, &sp, ss, 4);
  if (ts.rc) return ts.rc;
  const bool al = ts.wide;
  a.C = d->channels;
  a.N = d->inner;
  a.cols_all = d->batch * d->channels * d->inner;
  const int V = al ? 16 / ts.size : 1;
  const int64_t blocks = (a.cols_all / V + 255) / 256;
  if (!fits_launch((double)blocks, 256))
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: more columns than one launch takes");
  hipStream_t s = (hipStream_t)stream;
#define PT_STEP(F, T, V_) hipLaunchKernelGGL((k_scan_step<F, T, V_>), dim3((unsigned)blocks), dim3(256), 0, s, a, sp, ss)
#define PT_STEP_T(F)                                                                     \
  do {                                                                                   \
    if (d->dtype == PT_SCAN_F32) { if (al) PT_STEP(F, float, 4); else PT_STEP(F, float, 1); }        \
    else if (d->dtype == PT_SCAN_BF16) { if (al) PT_STEP(F, __bf16, 8); else PT_STEP(F, __bf16, 1); } \
    else { if (al) PT_STEP(F, _Float16, 8); else PT_STEP(F, _Float16, 1); }              \
  } while (0)
  if (d->form == PT_SCAN_LEAKY) PT_STEP_T(PT_SCAN_LEAKY);
  else PT_STEP_T(PT_SCAN_LSTM);
#undef PT_STEP_T
#undef PT_STEP
  return hipGetLastError() == hipSuccess ? 0 : fail(PT_SCAN_ERR_HIP, "scan: step launch failed");
}

}  // extern "C"
