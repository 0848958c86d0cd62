// pt_clip.hip — the global norm of many gradients, and clipping (include/pt_clip.h).
//
// Bound by memory: the norm reads every gradient once, the scaling reads it
// again and writes it.  The tensors' pointers travel in the kernel arguments
// (4 KB a launch: no copy to the device, nothing to keep alive), a tensor is cut
// into chunks of CHUNK elements, and a workgroup takes chunks id, id + grid, ...
// Every workgroup leaves one 64-bit partial; the scaling's workgroups each add
// all partials themselves, in the same order, which costs less than a launch
// between the two.  The scaling walks the chunks from the last to the first:
// what the norm read last is still in the card's cache.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <new>
#include <vector>

#include "pt_clip.h"

#ifndef PT_SRC_HASH
#define PT_SRC_HASH "unknown"
#endif

namespace {

thread_local char g_err[256] = "";

int fail(int code, const char* msg) {
  snprintf(g_err, sizeof(g_err), "%s", msg);
  return code;
}

constexpr int NT = 256;               // threads of a workgroup
constexpr int CHUNK = 8192;           // elements of a tensor that a workgroup takes at a time
constexpr int GRID = 1024;            // workgroups of a launch at most: 4 a compute unit
constexpr int64_t INLINE_PARTS = 4096;   // partials that every workgroup adds by itself
constexpr int64_t PIECE = (int64_t)1 << 28;   // elements of a table entry; larger tensors take several

// A launch's tensors, as many as 4 KB of kernel arguments hold: 12 bytes each
// where outputs are the gradients themselves (or there are none), else 20.
template <bool OUT> struct Table {
  static constexpr int MAX = OUT ? 192 : 320;
  const void* in[MAX];
  void* out[OUT ? MAX : 1];
  uint32_t n[MAX];                    // elements << 2 in 30 bits, type in the low two
  uint32_t out_f32[OUT ? MAX / 32 : 1];   // bit: the output is f32, whatever the gradient
  int count;
};
static_assert(sizeof(Table<false>) <= 3960 && sizeof(Table<true>) <= 3960, "kernel arguments of 4 KB");

// V elements in one access, at any alignment of their own.  A lane moves 16 bytes
// of the wider side at a time, so that a wave's access is one run of 1 KB (32
// bytes a lane leave every other 16 to the next access).
template <typename T, int V> using vecu = T __attribute__((ext_vector_type(V), aligned(sizeof(T))));

// Two partial results joined; a NaN stays.
template <int P> __device__ __forceinline__ double join(double a, double b) {
  if constexpr (P == PT_CLIP_INF) return a > b || a != a ? a : b;
  return a + b;
}
template <int P> __device__ __forceinline__ double term(double acc, float x) {
  if constexpr (P == PT_CLIP_L2) return __builtin_fma((double)x, (double)x, acc);
  if constexpr (P == PT_CLIP_L1) return acc + (double)__builtin_fabsf(x);
  const double v = (double)__builtin_fabsf(x);
  return acc > v || acc != acc ? acc : v;
}

// Join over the workgroup in a fixed order; every thread gets the result.
template <int P> __device__ double block_join(double v, double* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<P>(v, __shfl_xor(v, o));
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int k = 1; k < NT / 64; ++k) v = join<P>(v, red[k]);
  return v;
}

// First chunk of every tensor of the table, and the chunks of all (at [count]),
// in shared memory: a running sum by the first wave.
template <typename Tab> __device__ __forceinline__ void first_chunks(const Tab& t, uint32_t* first) {
  if (threadIdx.x < 64) {
    uint32_t base = 0;
    for (int k0 = 0; k0 < t.count; k0 += 64) {
      const int k = k0 + threadIdx.x;
      const uint32_t c = k < t.count ? ((t.n[k] >> 2) + CHUNK - 1) / CHUNK : 0;
      uint32_t s = c;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(s, o);
        if ((int)threadIdx.x >= o) s += v;
      }
      if (k < t.count) first[k] = base + s - c;
      base += __shfl(s, 63);
    }
    if (threadIdx.x == 0) first[t.count] = base;
  }
  __syncthreads();
}

// The tensor that chunk id belongs to (uniform over the workgroup).
__device__ __forceinline__ int tensor_of(const uint32_t* first, int count, uint32_t id) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= id) lo = mid; else hi = mid - 1;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

template <int P, typename T> __device__ __forceinline__ double chunk_norm(const T* p, uint32_t n, double acc) {
  constexpr int V = 16 / sizeof(T), U = CHUNK / (NT * V);
  vecu<T, V> v[U];
  if (n >= CHUNK) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *(const vecu<T, V>*)(p + (u * NT + threadIdx.x) * V);
  } else {                               // a tensor's end: one thread has a part of its V elements
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = (u * NT + threadIdx.x) * V;
      v[u] = (T)0.f;
      if (i + V <= n) {
        v[u] = *(const vecu<T, V>*)(p + i);
      } else if (i < n) {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (i + k < n) v[u][k] = p[i + k];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < V; ++k) acc = term<P>(acc, (float)v[u][k]);
  return acc;
}

// The partials.  Bound by memory: 335 million bf16 elements (671 MB) in 153 us, 4.4
// TB/s; 257 ragged tensors of three types (56 MB) in 16 us; 30 small ones in 5 us,
// which is the launch.  512 or 2048 workgroups, chunks of 4096 or 16384: the same or
// up to a tenth slower.
template <int P> __global__ __launch_bounds__(NT) void k_norm(Table<false> t, double* part) {
  __shared__ double red[NT / 64];
  __shared__ uint32_t first[Table<false>::MAX + 1];
  first_chunks(t, first);
  double acc = 0.0;
  const uint32_t total = first[t.count];
  for (uint32_t id = blockIdx.x; id < total; id += gridDim.x) {
    const int k = tensor_of(first, t.count, id);
    const uint32_t at = (id - first[k]) * CHUNK, n = (t.n[k] >> 2) - at, type = t.n[k] & 3;
    if (type == PT_CLIP_F32) acc = chunk_norm<P>((const float*)t.in[k] + at, n, acc);
    else if (type == PT_CLIP_BF16) acc = chunk_norm<P>((const __bf16*)t.in[k] + at, n, acc);
    else acc = chunk_norm<P>((const _Float16*)t.in[k] + at, n, acc);
  }
  acc = block_join<P>(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int P> __device__ double total_of(const double* part, int64_t parts, double* red) {
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < parts; i += NT) acc = join<P>(acc, part[i]);
  return block_join<P>(acc, red);
}
template <int P> __device__ __forceinline__ double root(double s) { return P == PT_CLIP_L2 ? sqrt(s) : s; }

// All partials to one (many of them), and to the norm where only that is asked for.
template <int P> __global__ __launch_bounds__(NT) void k_total(const double* part, int64_t parts, double* one, float* norm) {
  __shared__ double red[NT / 64];
  const double s = total_of<P>(part, parts, red);
  if (threadIdx.x == 0) {
    if (one) *one = s;
    if (norm) *norm = (float)root<P>(s);
  }
}

template <typename T, typename O>
__device__ __forceinline__ void chunk_scale(const T* p, O* o, uint32_t n, double k) {
  constexpr int V = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O)), U = CHUNK / (NT * V);
  auto times = [k](T x) { return (O)(float)((double)(float)x * k); };
  if (n >= CHUNK) {
    vecu<T, V> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *(const vecu<T, V>*)(p + (u * NT + threadIdx.x) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vecu<O, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r[j] = times(v[u][j]);
      *(vecu<O, V>*)(o + (u * NT + threadIdx.x) * V) = r;
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = (u * NT + threadIdx.x) * V;
      if (i + V <= n) {
        const vecu<T, V> v = *(const vecu<T, V>*)(p + i);
        vecu<O, V> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = times(v[j]);
        *(vecu<O, V>*)(o + i) = r;
      } else if (i < n) {
        for (uint32_t j = i; j < n; ++j) o[j] = times(p[j]);
      }
    }
  }
}

// The scaling: 335 million bf16 gradients into f32 (2.0 GB, two launches) in 373 us,
// 5.4 TB/s.  (With stores past the caches the whole call took 698 us instead of 567.)
template <int P, bool OUT>
__global__ __launch_bounds__(NT) void k_scale(Table<OUT> t, const double* part, int64_t parts, double max_norm,
                                              float* norm) {
  __shared__ double red[NT / 64];
  __shared__ uint32_t first[Table<OUT>::MAX + 1];
  const double n = root<P>(total_of<P>(part, parts, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double q = max_norm / (n + 1e-6);
  if (!OUT && q >= 1.0) return;                          // k = 1 in place: nothing changes
  // The product is taken in 64 bits and rounded once: k is far below f32's range
  // when the norm is far above it.  (A NaN goes through.)
  const double k = q >= 1.0 ? 1.0 : q;
  first_chunks(t, first);
  const uint32_t total = first[t.count];
  for (uint32_t r = blockIdx.x; r < total; r += gridDim.x) {
    const uint32_t id = total - 1 - r;
    const int i = tensor_of(first, t.count, id);
    const uint32_t at = (id - first[i]) * CHUNK, left = (t.n[i] >> 2) - at, type = t.n[i] & 3;
    const void* p = t.in[i];
    void* o = OUT ? t.out[OUT ? i : 0] : (void*)p;
    const bool wide = OUT && (t.out_f32[OUT ? i / 32 : 0] >> (i % 32) & 1);
    if (type == PT_CLIP_F32) {
      chunk_scale((const float*)p + at, (float*)o + at, left, k);
    } else if (type == PT_CLIP_BF16) {
      if (wide) chunk_scale((const __bf16*)p + at, (float*)o + at, left, k);
      else chunk_scale((const __bf16*)p + at, (__bf16*)o + at, left, k);
    } else {
      if (wide) chunk_scale((const _Float16*)p + at, (float*)o + at, left, k);
      else chunk_scale((const _Float16*)p + at, (_Float16*)o + at, left, k);
    }
  }
}

// ------------------------------------------------------------------ host

int size_of(int type) { return type == PT_CLIP_F32 ? 4 : 2; }

// Where a walk over the tensors stands: tensor, and element in it.
struct At {
  int64_t i = 0, e = 0;
};

// The next launch's tensors from `at` on, which moves behind them: their chunks.
template <bool OUT> uint32_t next_table(const pt_clip_tensor* t, int64_t count, At& at, Table<OUT>& tab) {
  uint32_t chunks = 0;
  tab.count = 0;
  if (OUT) std::fill(std::begin(tab.out_f32), std::end(tab.out_f32), 0u);
  while (at.i < count && tab.count < Table<OUT>::MAX) {
    const pt_clip_tensor& x = t[at.i];
    const int64_t n = std::min(x.n - at.e, PIECE);
    if (n > 0) {
      const int k = tab.count++;
      tab.in[k] = (const char*)x.grad + at.e * size_of(x.grad_type);
      tab.n[k] = (uint32_t)n << 2 | (uint32_t)x.grad_type;
      if (OUT) {
        tab.out[OUT ? k : 0] = (char*)x.out + at.e * size_of(x.out_type);
        if (x.out_type == PT_CLIP_F32) tab.out_f32[OUT ? k / 32 : 0] |= 1u << (k % 32);
      }
      chunks += (uint32_t)((n + CHUNK - 1) / CHUNK);
      at.e += n;
    }
    if (at.e >= x.n) at = At{at.i + 1, 0};
  }
  return chunks;
}

unsigned grid_of(uint32_t chunks) { return std::min<uint32_t>(chunks, GRID); }

int check(const pt_clip_tensor* t, int64_t count, bool out) {
  if (count < 0 || (count > 0 && !t)) return fail(PT_CLIP_ERR_ARG, "clip: null tensor list");
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n < 0) return fail(PT_CLIP_ERR_ARG, "clip: a tensor's size is negative");
    if (t[i].n == 0) continue;
    if (t[i].n > ((int64_t)1 << 44)) return fail(PT_CLIP_ERR_UNSUPPORTED, "clip: a tensor has more than 2^44 elements");
    if (t[i].grad_type < PT_CLIP_F32 || t[i].grad_type > PT_CLIP_F16)
      return fail(PT_CLIP_ERR_ARG, "clip: unknown gradient type");
    if (!t[i].grad || (out && !t[i].out)) return fail(PT_CLIP_ERR_ARG, "clip: null pointer");
    if ((uintptr_t)t[i].grad % size_of(t[i].grad_type))
      return fail(PT_CLIP_ERR_ARG, "clip: a tensor is not aligned to its elements");
    if (!out) continue;
    if (t[i].out_type != t[i].grad_type && t[i].out_type != PT_CLIP_F32)
      return fail(PT_CLIP_ERR_ARG, "clip: an output has its gradient's type or f32");
    if ((uintptr_t)t[i].out % size_of(t[i].out_type))
      return fail(PT_CLIP_ERR_ARG, "clip: a tensor is not aligned to its elements");
  }
  return 0;
}

// Written memory may be shared with nothing but its own gradient, in place:
// workgroups scale their chunks in no order.
int check_overlap(const pt_clip_tensor* t, int64_t count) {
  struct Range { uintptr_t lo, hi; bool written; };
  std::vector<Range> r;
  r.reserve((size_t)count * 2);
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n == 0) continue;
    const uintptr_t a = (uintptr_t)t[i].grad, o = (uintptr_t)t[i].out;
    const bool place = a == o && t[i].grad_type == t[i].out_type;
    if (!place) r.push_back({a, a + (uintptr_t)t[i].n * size_of(t[i].grad_type), false});
    r.push_back({o, o + (uintptr_t)t[i].n * size_of(t[i].out_type), true});
  }
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.lo < y.lo; });
  uintptr_t any = 0, written = 0;
  for (const Range& x : r) {
    if (x.lo < (x.written ? any : written))
      return fail(PT_CLIP_ERR_ARG, "clip: an output shares memory with another tensor of the call");
    any = std::max(any, x.hi);
    if (x.written) written = std::max(written, x.hi);
  }
  return 0;
}

int64_t parts_of(const pt_clip_tensor* t, int64_t count) {
  Table<false> tab;
  int64_t parts = 0;
  for (At at; at.i < count;) parts += grid_of(next_table(t, count, at, tab));
  return parts;
}

// The scaling's launches, from the last tensors to the first.
template <int P, bool OUT>
void scale_all(const pt_clip_tensor* t, int64_t count, const double* part, int64_t parts, double max_norm, float* norm,
               hipStream_t s) {
  Table<OUT> tab;
  std::vector<At> starts;
  for (At at; at.i < count;) {
    starts.push_back(at);
    next_table(t, count, at, tab);
  }
  for (size_t k = starts.size(); k-- > 0;) {
    At at = starts[k];
    const unsigned g = grid_of(next_table(t, count, at, tab));
    if (!g) continue;
    hipLaunchKernelGGL((k_scale<P, OUT>), dim3(g), dim3(NT), 0, s, tab, part, parts, max_norm, norm);
    norm = nullptr;                                      // written once
  }
}

template <int P>
int run(const pt_clip_tensor* t, int64_t count, bool scale, double max_norm, float* norm, double* part,
        hipStream_t s) {
  Table<false> tab;
  int64_t parts = 0;
  for (At at; at.i < count;) {
    const unsigned g = grid_of(next_table(t, count, at, tab));
    if (g) hipLaunchKernelGGL((k_norm<P>), dim3(g), dim3(NT), 0, s, tab, part + parts);
    parts += g;
  }
  const double* from = part;
  int64_t n = parts;
  if (!scale || parts == 0 || parts > INLINE_PARTS) {
    hipLaunchKernelGGL((k_total<P>), dim3(1), dim3(NT), 0, s, (const double*)part, parts, part + parts, norm);
    from = part + parts;
    n = 1;
    norm = nullptr;
  }
  if (scale && parts) {
    bool place = true;
    for (int64_t i = 0; i < count; ++i) place = place && (t[i].n == 0 || t[i].out == t[i].grad);
    if (place) scale_all<P, false>(t, count, from, n, max_norm, norm, s);
    else scale_all<P, true>(t, count, from, n, max_norm, norm, s);
  }
  return hipGetLastError() == hipSuccess ? 0 : fail(PT_CLIP_ERR_HIP, "clip: launch failed");
}

int run_p(const pt_clip_tensor* t, int64_t count, int norm_type, bool scale, double max_norm, float* norm,
          void* workspace, pt_clip_stream_t stream) {
  double* part = (double*)workspace;
  hipStream_t s = (hipStream_t)stream;
  if (!norm || !workspace) return fail(PT_CLIP_ERR_ARG, "clip: null pointer");
  switch (norm_type) {
    case PT_CLIP_INF: return run<PT_CLIP_INF>(t, count, scale, max_norm, norm, part, s);
    case PT_CLIP_L1: return run<PT_CLIP_L1>(t, count, scale, max_norm, norm, part, s);
    case PT_CLIP_L2: return run<PT_CLIP_L2>(t, count, scale, max_norm, norm, part, s);
    default: return fail(PT_CLIP_ERR_ARG, "clip: the norm is 1, 2 or inf");
  }
}

}  // namespace

extern "C" {

const char* pt_clip_last_error(void) { return g_err; }
const char* pt_clip_version(void) { return "pt_clip 0.1 gfx950 src " PT_SRC_HASH; }

size_t pt_clip_workspace_bytes(const pt_clip_tensor* t, int64_t count) {
  if (check(t, count, false)) return 0;
  return (size_t)(parts_of(t, count) + 1) * sizeof(double);
}

int pt_clip_norm(const pt_clip_tensor* t, int64_t count, int norm_type, float* norm, void* workspace,
                 pt_clip_stream_t stream) {
  if (int rc = check(t, count, false)) return rc;
  try {
    return run_p(t, count, norm_type, false, 0.0, norm, workspace, stream);
  } catch (const std::bad_alloc&) {
    return fail(PT_CLIP_ERR_HIP, "clip: out of host memory");
  }
}

int pt_clip_grads(const pt_clip_tensor* t, int64_t count, int norm_type, double max_norm, float* norm,
                  void* workspace, pt_clip_stream_t stream) {
  if (int rc = check(t, count, true)) return rc;
  if (!(max_norm >= 0.0)) return fail(PT_CLIP_ERR_ARG, "clip: max_norm must be >= 0");
  try {
    if (int rc = check_overlap(t, count)) return rc;
    return run_p(t, count, norm_type, true, max_norm, norm, workspace, stream);
  } catch (const std::bad_alloc&) {
    return fail(PT_CLIP_ERR_HIP, "clip: out of host memory");
  }
}

}  // extern "C"
