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
// Layout.  A lane owns V neighbouring columns (channel, inner), so every load
// of a wave is 64 V neighbouring elements of one step.  Where the columns do
// not fill the card the time axis is also cut over workgroups (`segs`): a
// first launch reduces each segment to (P, q), and the second starts each
// segment from the composition of those before it.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

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

constexpr int64_t MAX_SEGS = 64;
constexpr int SPLIT_W = 16;      // waves of a workgroup when the time axis is cut over workgroups

struct View {
  char* p;
  int64_t sb, sc, st;      // element strides
};

struct Args {
  View x[4], y, dx[4];     // y: the output, or dy in the backward
  const float* h0;
  const int64_t* len;
  float* h_last;
  float* c_last;
  const float* d_h_last;
  const float* d_c_last;
  float* d_h0;
  float* saved;            // [chunk][B][C N]: the state before a chunk (chunk 0: h0)
  float* agg;              // [segment][B][C N] pairs (P, q)
  int64_t T, cols_all;     // steps; B C N
  int64_t C, N;
  int64_t cg, groups;      // channels per column group, groups per batch row
  int64_t outer;           // B groups
  int64_t seg_steps;       // a multiple of the chunk
  int tiles, segs;
};

template <typename T, int V> using vec = T __attribute__((ext_vector_type(V)));

// e^-x for x >= 0.  ACC (f32 data): the product x log2(e) is carried in two
// parts, which keeps the error at an ulp for large x too; for 16-bit data the
// single product's error (x 2^-24 relative) is far below the data's step.
template <bool ACC> __device__ __forceinline__ float exp_minus(float x) {
  constexpr float L2E = 1.44269502f, L2E_LO = 1.92596303e-8f, LN2 = 0.693147182f;
  if constexpr (ACC) {
    x = x > 104.f ? 104.f : x;                 // (inf would make the low part NaN; NaN stays)
    const float t = x * L2E;
    const float lo = __builtin_fmaf(x, L2E_LO, __builtin_fmaf(x, L2E, -t));
    const float r = __builtin_amdgcn_exp2f(-t);
    return __builtin_fmaf(r, -lo * LN2, r);
  } else {
    return __builtin_amdgcn_exp2f(-x * L2E);
  }
}

template <bool ACC> __device__ __forceinline__ float recip(float d) {
  const float r = __builtin_amdgcn_rcpf(d);
  if constexpr (ACC) return __builtin_fmaf(r, __builtin_fmaf(-d, r, 1.f), r);
  return r;
}

// s(x) and s(-x), both to full relative accuracy (1 - s(x) would cancel).
template <bool ACC> __device__ __forceinline__ void logistic(float x, float& s, float& sm) {
  const float e = exp_minus<ACC>(__builtin_fabsf(x));
  const float big = recip<ACC>(1.f + e), small = e * big;
  s = x >= 0.f ? big : small;
  sm = x >= 0.f ? small : big;
}

// tanh(x) and its derivative 4 e / (1 + e)^2, e = exp(-2|x|).  f32 data: the
// odd series below 0.35 (next term 2e-9 relative), where 1 - e would cancel.
template <bool ACC> __device__ __forceinline__ float tanh_d(float x, float& d) {
  const float ax = __builtin_fabsf(x);
  const float e = exp_minus<ACC>(2.f * ax), r = recip<ACC>(1.f + e);
  d = 4.f * e * r * r;
  float t = __builtin_copysignf((1.f - e) * r, x);
  if constexpr (ACC) {
    const float q = x * x;
    float p = -1382.f / 155925.f;
    p = __builtin_fmaf(p, q, 62.f / 2835.f);
    p = __builtin_fmaf(p, q, -17.f / 315.f);
    p = __builtin_fmaf(p, q, 2.f / 15.f);
    p = __builtin_fmaf(p, q, -1.f / 3.f);
    t = ax < 0.35f ? __builtin_fmaf(x * q, p, x) : t;
  }
  return t;
}

// Shared memory between the waves of a workgroup: order LDS traffic alone, so
// that the loads in flight for the next chunk are not waited for.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Where a workgroup works: column tile, row, segment; and a lane's columns.
template <int V> struct Where {
  int seg, lane, wave;
  int64_t b, row, end;       // batch row; its end; index of the group's first channel in [B C]
  bool on;                   // this lane's columns exist
  int64_t state;             // index of this lane's first column in [B][C][N]
  uint32_t off_c, off_n;     // channel in the group, position in the inner axis

  __device__ __forceinline__ Where(const Args& a) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t id = blockIdx.x;            // the host keeps the grid below 2^31
    const uint32_t tile = id % (uint32_t)a.tiles;
    id /= (uint32_t)a.tiles;
    const uint32_t o = id % (uint32_t)a.outer;
    seg = (int)(id / (uint32_t)a.outer);
    const uint32_t br = o / (uint32_t)a.groups;
    const int64_t g = o - br * (uint32_t)a.groups;
    b = br;
    row = b * a.C + g * a.cg;
    const uint32_t cols = (uint32_t)(a.cg * a.N);
    uint32_t j = tile * 64 * V + lane * V;
    on = j < cols;
    j = on ? j : 0;          // an idle lane reads column 0 and stores nothing
    off_c = a.cg == 1 ? 0 : j / (uint32_t)a.N;
    off_n = j - off_c * (uint32_t)a.N;
    state = row * a.N + j;
    end = a.T;
    if (a.len) {
      const int64_t n = a.len[b];
      end = n < 0 ? 0 : n < a.T ? n : a.T;
    }
  }
  // byte offset of this lane within a step of the view (fits 32 bits: the host checks)
  template <typename T> __device__ __forceinline__ uint32_t lane_off(const View& v) const {
    return (uint32_t)((off_c * v.sc + off_n) * (int64_t)sizeof(T));
  }
  // the group's base at step 0
  template <typename T> __device__ __forceinline__ char* base(const Args& a, const View& v) const {
    const int64_t c0 = row - b * a.C;
    return v.p + (b * v.sb + c0 * v.sc) * (int64_t)sizeof(T);
  }
};

template <typename T, int V>
__device__ __forceinline__ vec<T, V> load(const char* base, uint32_t off) {
  return *(const vec<T, V>*)(base + off);
}
template <typename T, int V>
__device__ __forceinline__ void store(char* base, uint32_t off, vec<T, V> v) {
  *(vec<T, V>*)(base + off) = v;
}

// L steps from t0 of one view; steps at or behind lim are not read.
template <typename T, int V, int L>
__device__ __forceinline__ void load_steps(vec<T, V> (&r)[L], const char* base, int64_t st_bytes, uint32_t off,
                                           int64_t t0, int64_t lim) {
  const char* p = base + t0 * st_bytes;
  if (t0 + L <= lim) {
#pragma unroll
    for (int l = 0; l < L; ++l) r[l] = load<T, V>(p + l * st_bytes, off);
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      r[l] = 0;
      if (t0 + l < lim) r[l] = load<T, V>(p + l * st_bytes, off);
    }
  }
}

template <int FORM> constexpr int gates_of() { return FORM == PT_SCAN_LEAKY ? 2 : 4; }
// steps of one wave in a chunk: as many as two sets of the gates fit in registers
template <int FORM> constexpr int steps_of() { return FORM == PT_SCAN_LEAKY ? 8 : 4; }

// Compose the waves' (P, q) of one chunk: the state before this wave's steps
// from the one before the chunk, which becomes the one after it.
template <int W, int V>
__device__ __forceinline__ void compose(const float (&pq)[W][V][2][64], int wave, int lane, float (&carry)[V],
                                        float (&mine)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float c = carry[v];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      mine[v] = k == wave ? c : mine[v];
      c = __builtin_fmaf(pq[k][v][0][lane], c, pq[k][v][1][lane]);
    }
    carry[v] = c;
  }
}

// The state before segment `seg`.
template <int V>
__device__ __forceinline__ void start_state(const Args& a, const Where<V>& w, float (&c)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = a.h0 ? a.h0[w.state + v] : 0.f;
  for (int s = 0; s < w.seg; ++s) {
    const float* p = a.agg + 2 * (s * a.cols_all + w.state);
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = __builtin_fmaf(p[2 * v], c[v], p[2 * v + 1]);
  }
}

// Forward.  AGG: reduce a segment to (P, q) only.
template <int FORM, typename T, int V, int W, bool AGG>
__global__ __launch_bounds__(64 * W) void k_scan_fwd(Args a) {
  static_assert(W > 1 || !AGG, "one wave never splits the time axis over workgroups");
  constexpr int G = gates_of<FORM>(), L = steps_of<FORM>(), CH = W * L;
  constexpr bool ACC = sizeof(T) == 4;
  constexpr int GA = FORM == PT_SCAN_LEAKY ? 2 : 3;      // the gates that make a and b
  __shared__ float pq[2][W][V][2][64];   // two sets in turn, as in the backward
  const Where<V> w(a);
  const int64_t t_beg = w.seg * a.seg_steps;
  const int64_t t_end = t_beg + a.seg_steps < a.T ? t_beg + a.seg_steps : a.T;
  const int64_t lim = w.end < t_end ? w.end : t_end;
  const bool seq = !AGG && a.y.p != nullptr;

  float carry[V], prod[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { carry[v] = 0.f; prod[v] = 1.f; }
  if constexpr (!AGG) start_state<V>(a, w, carry);

  const char* xb[G];
  uint32_t xo[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    xb[g] = w.template base<T>(a, a.x[g]);
    xo[g] = w.template lane_off<T>(a.x[g]);
  }
  char* yb = seq ? w.template base<T>(a, a.y) : nullptr;
  const uint32_t yo = seq ? w.template lane_off<T>(a.y) : 0;
  const int64_t ys = a.y.st * (int64_t)sizeof(T);

  vec<T, V> raw[G][L];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int g = 0; g < GA; ++g)
      load_steps<T, V, L>(raw[g], xb[g], a.x[g].st * (int64_t)sizeof(T), xo[g], t0, lim);
    if constexpr (!AGG && FORM == PT_SCAN_LSTM)      // o is wanted for y, or at the row's last step
      if (seq || (t0 < w.end && w.end <= t0 + L))
        load_steps<T, V, L>(raw[3], xb[3], a.x[3].st * (int64_t)sizeof(T), xo[3], t0, lim);
  };
  fetch(t_beg + w.wave * L);

  int par = 0;
  for (int64_t t = t_beg; t < t_end; t += CH) {
    const int64_t t0 = t + w.wave * L;
    if (t >= lim) {                                   // the whole chunk is behind the row's end
      if (!seq) break;
      if (w.on) {
#pragma unroll
        for (int l = 0; l < L; ++l)
          if (t0 + l < t_end) store<T, V>(yb + (t0 + l) * ys, yo, (vec<T, V>)(0));
      }
      continue;
    }
    if constexpr (!AGG)
      if (a.saved && t > 0 && w.wave == 0 && w.on) {
        float* s = a.saved + (t / CH - 1) * a.cols_all + w.state;
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = carry[v];
      }
    float A[L][V], B[L][V];
    vec<T, V> o[L];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const bool live = t0 + l < lim;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s, sm, d;
        if constexpr (FORM == PT_SCAN_LEAKY) {
          logistic<ACC>((float)raw[0][l][v], s, sm);
          A[l][v] = live ? sm : 1.f;
          B[l][v] = live ? s * (float)raw[1][l][v] : 0.f;
        } else {
          logistic<ACC>((float)raw[1][l][v], s, sm);
          A[l][v] = live ? s : 1.f;
          logistic<ACC>((float)raw[0][l][v], s, sm);
          B[l][v] = live ? s * tanh_d<ACC>((float)raw[2][l][v], d) : 0.f;
        }
      }
      if constexpr (!AGG && FORM == PT_SCAN_LSTM) o[l] = raw[3][l];
    }
    if (t + CH < lim) fetch(t0 + CH);

    float cin[V];
    if constexpr (W == 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) cin[v] = carry[v];
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float p = 1.f, q = 0.f;
#pragma unroll
        for (int l = 0; l < L; ++l) {
          q = __builtin_fmaf(A[l][v], q, B[l][v]);
          p *= A[l][v];
        }
        pq[par][w.wave][v][0][w.lane] = p;
        pq[par][w.wave][v][1][w.lane] = q;
      }
      lds_barrier();
      compose<W, V>(pq[par], w.wave, w.lane, carry, cin);
      if constexpr (AGG) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < W; ++k) prod[v] *= pq[par][k][v][0][w.lane];
      }
      par ^= 1;
    }
    if constexpr (AGG) continue;

    const bool has_last = t0 < w.end && w.end <= t0 + L;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      vec<T, V> out;
      float yl[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        cin[v] = __builtin_fmaf(A[l][v], cin[v], B[l][v]);
        yl[v] = cin[v];
      }
      if constexpr (!AGG) {
        if constexpr (FORM == PT_SCAN_LSTM) {
          if (seq || has_last) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
              float s, sm, d;
              logistic<ACC>((float)o[l][v], s, sm);
              yl[v] = s * tanh_d<ACC>(cin[v], d);
            }
            if (t0 + l == w.end - 1 && a.h_last && w.on) {
#pragma unroll
              for (int v = 0; v < V; ++v) a.h_last[w.state + v] = yl[v];
            }
          }
        }
        if (seq && w.on && t0 + l < t_end) {
#pragma unroll
          for (int v = 0; v < V; ++v) out[v] = (T)(t0 + l < lim ? yl[v] : 0.f);
          store<T, V>(yb + (t0 + l) * ys, yo, out);
        }
      }
    }
    if constexpr (W == 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) carry[v] = cin[v];
    }
  }

  if (w.wave != 0 || !w.on) return;
  if constexpr (AGG) {
    float* p = a.agg + 2 * (w.seg * a.cols_all + w.state);
#pragma unroll
    for (int v = 0; v < V; ++v) { p[2 * v] = prod[v]; p[2 * v + 1] = carry[v]; }
  } else if (w.seg == a.segs - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (a.c_last) a.c_last[w.state + v] = carry[v];
      if (a.h_last && FORM == PT_SCAN_LEAKY) a.h_last[w.state + v] = carry[v];
      if (a.h_last && FORM == PT_SCAN_LSTM && w.end == 0) a.h_last[w.state + v] = 0.f;
    }
  }
}

// Backward.  AGG: reduce a segment, from zero at its far end, to (P, q) of the
// gradient that leaves it towards the past.
template <int FORM, typename T, int V, int W, bool AGG>
__global__ __launch_bounds__(64 * W) void k_scan_bwd(Args a) {
  constexpr int G = gates_of<FORM>(), L = steps_of<FORM>(), CH = W * L;
  constexpr bool ACC = sizeof(T) == 4;
  // Two sets, used in turn: a wave writes a set again only behind a barrier that
  // every wave reaches after its last read of it, so one barrier an exchange does.
  __shared__ float pq[2][W][V][2][64];   // forward (P, q)
  __shared__ float gq[2][W][V][64];      // backward q (its P is the same)
  int par = 0;
  const Where<V> w(a);
  const int seg = AGG ? w.seg + 1 : w.seg;             // nothing is behind segment 0
  const int64_t t_beg = seg * a.seg_steps;
  const int64_t t_end = t_beg + a.seg_steps < a.T ? t_beg + a.seg_steps : a.T;
  const int64_t lim = w.end < t_end ? w.end : t_end;
  const bool has_dy = a.y.p != nullptr;

  float carry[V], prod[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { carry[v] = 0.f; prod[v] = 1.f; }
  if constexpr (!AGG) {
    const float* end = FORM == PT_SCAN_LEAKY ? a.d_h_last : a.d_c_last;
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = end ? end[w.state + v] : 0.f;
    for (int s = a.segs - 1; s > seg; --s) {
      const float* p = a.agg + 2 * ((s - 1) * a.cols_all + w.state);
#pragma unroll
      for (int v = 0; v < V; ++v) carry[v] = __builtin_fmaf(p[2 * v], carry[v], p[2 * v + 1]);
    }
  }

  const char* xb[G];
  char* db[G];
  uint32_t xo[G], dof[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    xb[g] = w.template base<T>(a, a.x[g]);
    xo[g] = w.template lane_off<T>(a.x[g]);
    db[g] = AGG ? nullptr : w.template base<T>(a, a.dx[g]);
    dof[g] = AGG ? 0 : w.template lane_off<T>(a.dx[g]);
  }
  const char* yb = has_dy ? w.template base<T>(a, a.y) : nullptr;
  const uint32_t yo = has_dy ? w.template lane_off<T>(a.y) : 0;

  vec<T, V> raw[G][L], rdy[L];
  float nst[V];                                         // the state before the fetched chunk
  auto fetch = [&](int64_t t) {
    const int64_t t0 = t + w.wave * L;
#pragma unroll
    for (int g = 0; g < G; ++g)
      load_steps<T, V, L>(raw[g], xb[g], a.x[g].st * (int64_t)sizeof(T), xo[g], t0, lim);
    if (has_dy)
      load_steps<T, V, L>(rdy, yb, a.y.st * (int64_t)sizeof(T), yo, t0, lim);
    const float* s = t > 0 ? a.saved + (t / CH - 1) * a.cols_all : a.h0;
#pragma unroll
    for (int v = 0; v < V; ++v) nst[v] = s ? s[w.state + v] : 0.f;
  };
#pragma unroll
  for (int l = 0; l < L; ++l) rdy[l] = 0;

  // chunks from the last to the first; those behind the row's end only clear dx
  int64_t t = t_beg + (t_end - 1 - t_beg) / CH * CH;
  for (; t >= t_beg && t >= lim; t -= CH) {
    if constexpr (!AGG) {
      if (w.on)
#pragma unroll
        for (int l = 0; l < L; ++l) {
          const int64_t tt = t + w.wave * L + l;
          if (tt < t_end)
#pragma unroll
            for (int g = 0; g < G; ++g)
              store<T, V>(db[g] + tt * a.dx[g].st * (int64_t)sizeof(T), dof[g], (vec<T, V>)(0));
        }
    }
  }
  if (t >= t_beg) fetch(t);
  for (; t >= t_beg; t -= CH) {
    const int64_t t0 = t + w.wave * L;
    float A[L][V], B[L][V], D[L][V];                    // a; b, then the state before the step; dy
    float K0[L][V], K1[L][V], K2[L][V];                 // what the gradients are made of
    float O[L][V], OD[L][V];                            // lstm: s(o), s(o) s(-o)
    float st[V];
#pragma unroll
    for (int v = 0; v < V; ++v) st[v] = nst[v];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const bool live = t0 + l < lim;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float s, sm, d;
        D[l][v] = live ? (float)rdy[l][v] : 0.f;
        if constexpr (FORM == PT_SCAN_LEAKY) {
          const float n = (float)raw[1][l][v];
          logistic<ACC>((float)raw[0][l][v], s, sm);
          A[l][v] = live ? sm : 1.f;
          B[l][v] = live ? s * n : 0.f;
          K0[l][v] = n;
          K1[l][v] = s;
        } else {
          logistic<ACC>((float)raw[1][l][v], s, sm);
          A[l][v] = live ? s : 1.f;
          K1[l][v] = s * sm;                            // d f
          logistic<ACC>((float)raw[0][l][v], s, sm);
          const float th = tanh_d<ACC>((float)raw[2][l][v], d);
          B[l][v] = live ? s * th : 0.f;
          K0[l][v] = th * s * sm;                       // d i
          K2[l][v] = s * d;                             // d n
          logistic<ACC>((float)raw[3][l][v], s, sm);
          O[l][v] = s;
          OD[l][v] = s * sm;
          if (a.d_h_last && t0 + l == w.end - 1) D[l][v] += a.d_h_last[w.state + v];
        }
      }
    }
    if (t - CH >= t_beg) fetch(t - CH);

    float cin[V], gin[V];
    if constexpr (W > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float p = 1.f, q = 0.f, g = 0.f;
#pragma unroll
        for (int l = 0; l < L; ++l) {
          q = __builtin_fmaf(A[l][v], q, B[l][v]);
          p *= A[l][v];
        }
        pq[par][w.wave][v][0][w.lane] = p;
        pq[par][w.wave][v][1][w.lane] = q;
        if constexpr (FORM == PT_SCAN_LEAKY) {          // y = h: dy needs no state
#pragma unroll
          for (int l = L - 1; l >= 0; --l) g = A[l][v] * (D[l][v] + g);
          gq[par][w.wave][v][w.lane] = g;
        }
      }
      lds_barrier();
      compose<W, V>(pq[par], w.wave, w.lane, st, cin);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) cin[v] = st[v];
    }

    // the states, forward; B becomes the state before each step
#pragma unroll
    for (int l = 0; l < L; ++l) {
      vec<T, V> dO;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float h = __builtin_fmaf(A[l][v], cin[v], B[l][v]);
        B[l][v] = cin[v];
        cin[v] = h;
        if constexpr (FORM == PT_SCAN_LSTM) {
          float d;
          const float th = tanh_d<ACC>(h, d);
          dO[v] = (T)(t0 + l < lim ? D[l][v] * th * OD[l][v] : 0.f);
          D[l][v] *= O[l][v] * d;
        }
      }
      if constexpr (FORM == PT_SCAN_LSTM && !AGG)
        if (w.on && t0 + l < t_end)
          store<T, V>(db[3] + (t0 + l) * a.dx[3].st * (int64_t)sizeof(T), dof[3], dO);
    }
    if constexpr (W > 1 && FORM == PT_SCAN_LSTM) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float g = 0.f;
#pragma unroll
        for (int l = L - 1; l >= 0; --l) g = A[l][v] * (D[l][v] + g);
        gq[par][w.wave][v][w.lane] = g;
      }
      lds_barrier();
    }
    if constexpr (W > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float c = carry[v];
#pragma unroll
        for (int k = W - 1; k >= 0; --k) {
          gin[v] = k == w.wave ? c : gin[v];
          const float p = pq[par][k][v][0][w.lane];
          if constexpr (AGG) prod[v] *= p;
          c = __builtin_fmaf(p, c, gq[par][k][v][w.lane]);
        }
        carry[v] = c;
      }
      par ^= 1;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) gin[v] = carry[v];
    }
    if constexpr (AGG) continue;

#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      vec<T, V> out[3];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float g = D[l][v] + gin[v];
        const bool live = t0 + l < lim;
        if constexpr (FORM == PT_SCAN_LEAKY) {
          const float gs = g * K1[l][v];
          out[0][v] = (T)(live ? gs * A[l][v] * (K0[l][v] - B[l][v]) : 0.f);
          out[1][v] = (T)(live ? gs : 0.f);
        } else {
          out[0][v] = (T)(live ? g * K0[l][v] : 0.f);
          out[1][v] = (T)(live ? g * B[l][v] * K1[l][v] : 0.f);
          out[2][v] = (T)(live ? g * K2[l][v] : 0.f);
        }
        gin[v] = A[l][v] * g;
      }
      if constexpr (!AGG)
        if (w.on && t0 + l < t_end) {
#pragma unroll
          for (int g = 0; g < G - (FORM == PT_SCAN_LSTM); ++g)
            store<T, V>(db[g] + (t0 + l) * a.dx[g].st * (int64_t)sizeof(T), dof[g], out[g]);
        }
    }
    if constexpr (W == 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) carry[v] = gin[v];
    }
  }

  if (w.wave != 0 || !w.on) return;
  if constexpr (AGG) {
    float* p = a.agg + 2 * ((int64_t)w.seg * a.cols_all + w.state);
#pragma unroll
    for (int v = 0; v < V; ++v) { p[2 * v] = prod[v]; p[2 * v + 1] = carry[v]; }
  } else if (seg == 0 && a.d_h0) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.d_h0[w.state + v] = carry[v];
  }
}

// One step: element-wise, one lane per V columns.
template <int FORM, typename T, int V>
__global__ __launch_bounds__(256) void k_scan_step(Args a, View state) {
  constexpr int G = gates_of<FORM>();
  constexpr bool ACC = sizeof(T) == 4;
  const int64_t cols = a.C * a.N;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= a.cols_all) return;
  const int64_t b = i / cols, j = i - b * cols;
  const int64_t c = a.C == 1 ? 0 : j / a.N, n = j - c * a.N;
  auto at = [&](const View& v) { return b * v.sb + c * v.sc + n; };
  vec<T, V> x[G], out;
#pragma unroll
  for (int g = 0; g < G; ++g) x[g] = *((const vec<T, V>*)((const T*)a.x[g].p + at(a.x[g])));
  float* sp = (float*)state.p + at(state);
  vec<float, V> h = *(const vec<float, V>*)sp;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s, sm, d;
    if constexpr (FORM == PT_SCAN_LEAKY) {
      logistic<ACC>((float)x[0][v], s, sm);
      h[v] = __builtin_fmaf(sm, h[v], s * (float)x[1][v]);
      out[v] = (T)h[v];
    } else {
      float f, i_, o;
      logistic<ACC>((float)x[1][v], f, sm);
      logistic<ACC>((float)x[0][v], i_, sm);
      logistic<ACC>((float)x[3][v], o, sm);
      h[v] = __builtin_fmaf(f, h[v], i_ * tanh_d<ACC>((float)x[2][v], d));
      out[v] = (T)(o * tanh_d<ACC>(h[v], d));
    }
  }
  *(vec<float, V>*)sp = h;
  *((vec<T, V>*)((T*)a.y.p + at(a.y))) = out;
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
  const int64_t big = (int64_t)1 << 40;
  if (d->batch > big || d->channels > big || d->steps > big || d->inner > big ||
      (double)d->batch * (double)d->channels * (double)d->inner * (double)d->steps > 1e15)
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: more elements than any device holds");
  if (d->inner >= ((int64_t)1 << 29))
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: inner must be below 2^29");
  return 0;
}

// How a shape is cut; from the descriptor alone, so that forward, backward and
// the size queries agree.
struct Plan {
  int W, L;
  int64_t chunk, nchunks, segs, seg_steps;
};

Plan plan_of(const pt_scan_desc* d) {
  Plan p;
  p.L = d->form == PT_SCAN_LEAKY ? 8 : 4;
  const int64_t wide = 64 * (d->dtype == PT_SCAN_F32 ? 1 : 2);
  const int64_t tiles = d->batch * ((d->channels * d->inner + wide - 1) / wide);
  p.W = d->steps <= p.L ? 1 : tiles >= 1024 || d->steps <= 4 * p.L ? 4 : SPLIT_W;
  p.chunk = (int64_t)p.W * p.L;
  p.nchunks = (d->steps + p.chunk - 1) / p.chunk;
  p.segs = 1;
  if (p.W == SPLIT_W && tiles < 512) {
    p.segs = (512 + tiles - 1) / tiles;
    if (p.segs > p.nchunks / 2) p.segs = p.nchunks / 2;
    if (p.segs > MAX_SEGS) p.segs = MAX_SEGS;
    if (p.segs < 1) p.segs = 1;
  }
  const int64_t per = (p.nchunks + p.segs - 1) / p.segs;
  p.segs = (p.nchunks + per - 1) / per;
  p.seg_steps = per * p.chunk;
  return p;
}

// Strides of axes of one element never count: 0, so that they cannot spoil the alignment.
pt_scan_view tidy(const pt_scan_desc* d, const pt_scan_view& v) {
  return pt_scan_view{v.data, d->batch == 1 ? 0 : v.sb, d->channels == 1 ? 0 : v.sc, d->steps == 1 ? 0 : v.st};
}
View view_of(const pt_scan_view& v) { return View{(char*)v.data, v.sb, v.sc, v.st}; }

// Both halves of the alignment rule: V elements of a lane are one load only if
// every stride and the base keep them aligned and V divides the inner axis.
bool aligned(const pt_scan_view& v, int V, int size) {
  return ((uintptr_t)v.data % (V * size)) == 0 && v.sb % V == 0 && v.sc % V == 0 && v.st % V == 0;
}

bool spans32(const pt_scan_desc* d, const pt_scan_view& v, int size) {
  const double s = ((double)(d->channels - 1) * (double)(v.sc < 0 ? -v.sc : v.sc) + (double)d->inner) * size;
  return v.sc >= 0 && s < 2147483648.0;
}

template <int FORM, typename T, int V, int W>
int launch_fwd(Args a, int64_t blocks, hipStream_t s) {
  if constexpr (W == SPLIT_W)
    if (a.segs > 1) {
      const int64_t n = blocks / a.segs * (a.segs - 1);
      hipLaunchKernelGGL((k_scan_fwd<FORM, T, V, W, true>), dim3((unsigned)n), dim3(64 * W), 0, s, a);
    }
  hipLaunchKernelGGL((k_scan_fwd<FORM, T, V, W, false>), dim3((unsigned)blocks), dim3(64 * W), 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : fail(PT_SCAN_ERR_HIP, "scan: forward launch failed");
}

template <int FORM, typename T, int V, int W>
int launch_bwd(Args a, int64_t blocks, hipStream_t s) {
  if constexpr (W == SPLIT_W)
    if (a.segs > 1) {
      const int64_t n = blocks / a.segs * (a.segs - 1);
      hipLaunchKernelGGL((k_scan_bwd<FORM, T, V, W, true>), dim3((unsigned)n), dim3(64 * W), 0, s, a);
    }
  hipLaunchKernelGGL((k_scan_bwd<FORM, T, V, W, false>), dim3((unsigned)blocks), dim3(64 * W), 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : fail(PT_SCAN_ERR_HIP, "scan: backward launch failed");
}

template <int FORM, typename T, int V>
int launch_w(const Plan& p, const Args& a, int64_t blocks, bool bwd, hipStream_t s) {
  switch (p.W) {
    case 1: return bwd ? launch_bwd<FORM, T, V, 1>(a, blocks, s) : launch_fwd<FORM, T, V, 1>(a, blocks, s);
    case 4: return bwd ? launch_bwd<FORM, T, V, 4>(a, blocks, s) : launch_fwd<FORM, T, V, 4>(a, blocks, s);
    default: return bwd ? launch_bwd<FORM, T, V, SPLIT_W>(a, blocks, s) : launch_fwd<FORM, T, V, SPLIT_W>(a, blocks, s);
  }
}

template <int FORM>
int launch_t(int dtype, int V, const Plan& p, const Args& a, int64_t blocks, bool bwd, hipStream_t s) {
  if (dtype == PT_SCAN_F32) return launch_w<FORM, float, 1>(p, a, blocks, bwd, s);
  if (dtype == PT_SCAN_BF16)
    return V == 2 ? launch_w<FORM, __bf16, 2>(p, a, blocks, bwd, s) : launch_w<FORM, __bf16, 1>(p, a, blocks, bwd, s);
  return V == 2 ? launch_w<FORM, _Float16, 2>(p, a, blocks, bwd, s) : launch_w<FORM, _Float16, 1>(p, a, blocks, bwd, s);
}

int run(const pt_scan_desc* d, const Plan& p, Args& a, const pt_scan_view* views, int nviews, bool bwd,
        hipStream_t s) {
  const int size = elem_size(d->dtype);
  int V = size == 4 || d->inner % 2 ? 1 : 2;
  bool grouped = true;
  for (int i = 0; i < nviews; ++i) {
    if (V > 1 && !aligned(views[i], V, size)) V = 1;
    if ((uintptr_t)views[i].data % size) return fail(PT_SCAN_ERR_ARG, "scan: a tensor is not aligned to its elements");
    if (!spans32(d, views[i], size)) grouped = false;
  }
  // Columns of one channel at a time where the inner axis fills whole tiles, or
  // where the channels of a step reach over more than a 32-bit offset.
  if (d->inner % (64 * V) == 0) grouped = false;
  if ((double)d->channels * (double)d->inner >= 2147483648.0) grouped = false;
  a.C = d->channels;
  a.N = d->inner;
  a.T = d->steps;
  a.cols_all = d->batch * d->channels * d->inner;
  a.cg = grouped ? d->channels : 1;
  a.groups = d->channels / a.cg;
  a.outer = d->batch * a.groups;
  a.segs = (int)p.segs;
  a.seg_steps = p.seg_steps;
  const int64_t tiles = (a.cg * a.N + 64 * V - 1) / (64 * V);
  a.tiles = (int)tiles;
  if ((double)tiles * (double)a.outer * (double)p.segs > 2147483647.0)
    return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: too many columns for one launch");
  const int64_t blocks = tiles * a.outer * p.segs;
  return d->form == PT_SCAN_LEAKY ? launch_t<PT_SCAN_LEAKY>(d->dtype, V, p, a, blocks, bwd, s)
                                  : launch_t<PT_SCAN_LSTM>(d->dtype, V, p, a, blocks, bwd, s);
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
  return (size_t)((p.segs - 1) * d->batch * d->channels * d->inner) * 2 * sizeof(float);
}

int pt_scan_forward(const pt_scan_desc* d, const pt_scan_view* x, const float* h0, const int64_t* lengths,
                    const pt_scan_view* y, float* h_last, float* c_last, void* saved, void* workspace,
                    pt_scan_stream_t stream) {
  if (int rc = check(d)) return rc;
  if (!x) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
  const Plan p = plan_of(d);
  Args a{};
  pt_scan_view views[5];
  int n = 0;
  for (int g = 0; g < gates(d->form); ++g) {
    if (!x[g].data) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
    a.x[g] = view_of(views[n++] = tidy(d, x[g]));
  }
  if (y && y->data) {
    a.y = view_of(views[n++] = tidy(d, *y));
  }
  if (p.segs > 1 && !workspace) return fail(PT_SCAN_ERR_ARG, "scan: this shape needs a workspace");
  a.h0 = h0; a.len = lengths; a.h_last = h_last; a.c_last = c_last;
  a.saved = p.nchunks > 1 ? (float*)saved : nullptr;
  a.agg = (float*)workspace;
  return run(d, p, a, views, n, false, (hipStream_t)stream);
}

int pt_scan_backward(const pt_scan_desc* d, const pt_scan_view* x, const float* h0, const int64_t* lengths,
                     const pt_scan_view* dy, const float* d_h_last, const float* d_c_last, const void* saved,
                     const pt_scan_view* dx, float* d_h0, void* workspace, pt_scan_stream_t stream) {
  if (int rc = check(d)) return rc;
  if (!x || !dx) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
  const Plan p = plan_of(d);
  Args a{};
  pt_scan_view views[9];
  int n = 0;
  for (int g = 0; g < gates(d->form); ++g) {
    if (!x[g].data || !dx[g].data) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
    a.x[g] = view_of(views[n++] = tidy(d, x[g]));
    a.dx[g] = view_of(views[n++] = tidy(d, dx[g]));
  }
  if (dy && dy->data) {
    a.y = view_of(views[n++] = tidy(d, *dy));
  }
  if (p.nchunks > 1 && !saved) return fail(PT_SCAN_ERR_ARG, "scan: the backward needs the forward's saved states");
  if (p.segs > 1 && !workspace) return fail(PT_SCAN_ERR_ARG, "scan: this shape needs a workspace");
  a.h0 = h0; a.len = lengths; a.d_h_last = d_h_last; a.d_c_last = d_c_last; a.d_h0 = d_h0;
  a.saved = (float*)saved;
  a.agg = (float*)workspace;
  return run(d, p, a, views, n, true, (hipStream_t)stream);
}

int pt_scan_step(const pt_scan_desc* d, const pt_scan_view* x, const pt_scan_view* state, const pt_scan_view* y,
                 pt_scan_stream_t stream) {
  if (int rc = check(d)) return rc;
  if (!x || !state || !y || !state->data || !y->data) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
  if (d->steps != 1) return fail(PT_SCAN_ERR_ARG, "scan: a step has steps = 1");
  const int size = elem_size(d->dtype), wide = 16 / size;
  Args a{};
  const pt_scan_view yv = tidy(d, *y), sv = tidy(d, *state);
  bool al = d->inner % wide == 0 && aligned(yv, wide, size) && aligned(sv, wide, 4);
  for (int g = 0; g < gates(d->form); ++g) {
    if (!x[g].data) return fail(PT_SCAN_ERR_ARG, "scan: null pointer");
    const pt_scan_view xv = tidy(d, x[g]);
    a.x[g] = view_of(xv);
    al = al && aligned(xv, wide, size);
    if ((uintptr_t)x[g].data % size) return fail(PT_SCAN_ERR_ARG, "scan: a tensor is not aligned to its elements");
  }
  if ((uintptr_t)y->data % size || (uintptr_t)state->data % 4)
    return fail(PT_SCAN_ERR_ARG, "scan: a tensor is not aligned to its elements");
  a.y = view_of(yv);
  a.C = d->channels;
  a.N = d->inner;
  a.cols_all = d->batch * d->channels * d->inner;
  const int V = al ? wide : 1;
  const int64_t blocks = (a.cols_all / V + 255) / 256;
  if (blocks > 2147483647) return fail(PT_SCAN_ERR_UNSUPPORTED, "scan: too many columns for one launch");
  const View st = view_of(sv);
  hipStream_t s = (hipStream_t)stream;
#define PT_STEP(F, T, V_) hipLaunchKernelGGL((k_scan_step<F, T, V_>), dim3((unsigned)blocks), dim3(256), 0, s, a, st)
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
