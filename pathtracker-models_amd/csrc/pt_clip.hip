// pt_clip.hip — the global norm of many gradients, and clipping (include/pt_clip.h).
//
// Bound by memory: the norm reads every gradient once, the scaling reads it
// again and writes it.  The tensors' pointers travel in the kernel arguments
// (TABLE of them a launch: no copy to the device, nothing to keep alive), a
// tensor is cut into chunks of CHUNK elements, and a workgroup takes chunks
// id, id + grid, ...  Every workgroup leaves one 64-bit partial; the scaling's
// workgroups each add all partials themselves, in the same order, which costs
// less than a launch between the two.  The scaling walks the chunks from the
// last to the first: what the norm read last is still in the card's cache.
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
constexpr int VEC = 8;                // elements of a thread at a time: 16 or 32 bytes
constexpr int UNROLL = 4;
constexpr int CHUNK = NT * VEC * UNROLL;
constexpr int TABLE = 96;             // tensors of a launch: 36 bytes each, under the 4 KB of arguments
constexpr int GRID = 1024;            // workgroups of a launch at most: 4 a compute unit
constexpr int64_t INLINE_PARTS = 4096;   // partials that every workgroup adds by itself

struct Table {
  const void* in[TABLE];
  void* out[TABLE];
  int64_t n[TABLE];
  uint32_t first[TABLE + 1];          // first chunk of each tensor
  uint8_t in_type[TABLE], out_type[TABLE];
  int count;
};

template <typename T> using vecu = T __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));

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

// The tensor that chunk id belongs to (uniform over the workgroup).
__device__ __forceinline__ int tensor_of(const Table& t, uint32_t id) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= id) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int P, typename T> __device__ __forceinline__ double chunk_norm(const T* p, int64_t n, double acc) {
  if (n >= CHUNK) {
    vecu<T> v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) v[u] = *(const vecu<T>*)(p + (u * NT + threadIdx.x) * VEC);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc = term<P>(acc, (float)v[u][k]);
  } else {
    for (int i = threadIdx.x; i < (int)n; i += NT) acc = term<P>(acc, (float)p[i]);
  }
  return acc;
}

template <int P> __global__ __launch_bounds__(NT) void k_norm(Table t, double* part) {
  __shared__ double red[NT / 64];
  double acc = 0.0;
  const uint32_t total = t.first[t.count];
  for (uint32_t id = blockIdx.x; id < total; id += gridDim.x) {
    const int k = tensor_of(t, id);
    const int64_t at = (int64_t)(id - t.first[k]) * CHUNK;
    const int64_t n = t.n[k] - at;
    if (t.in_type[k] == PT_CLIP_F32) acc = chunk_norm<P>((const float*)t.in[k] + at, n, acc);
    else if (t.in_type[k] == PT_CLIP_BF16) acc = chunk_norm<P>((const __bf16*)t.in[k] + at, n, acc);
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
__device__ __forceinline__ void chunk_scale(const T* p, O* o, int64_t n, double k) {
  if (n >= CHUNK) {
    vecu<T> v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) v[u] = *(const vecu<T>*)(p + (u * NT + threadIdx.x) * VEC);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      vecu<O> r;
#pragma unroll
      for (int j = 0; j < VEC; ++j) r[j] = (O)(float)((double)(float)v[u][j] * k);
      *(vecu<O>*)(o + (u * NT + threadIdx.x) * VEC) = r;
    }
  } else {
    for (int i = threadIdx.x; i < (int)n; i += NT) o[i] = (O)(float)((double)(float)p[i] * k);
  }
}

template <int P>
__global__ __launch_bounds__(NT) void k_scale(Table t, const double* part, int64_t parts, double max_norm, float* norm) {
  __shared__ double red[NT / 64];
  const double n = root<P>(total_of<P>(part, parts, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double q = max_norm / (n + 1e-6);
  // The product is taken in 64 bits and rounded once: k is far below f32's range
  // when the norm is far above it.  (A NaN goes through.)
  const double k = q >= 1.0 ? 1.0 : q;
  const uint32_t total = t.first[t.count];
  for (uint32_t r = blockIdx.x; r < total; r += gridDim.x) {
    const uint32_t id = total - 1 - r;
    const int i = tensor_of(t, id);
    if (q >= 1.0 && t.out[i] == t.in[i]) continue;       // k = 1 in place: nothing changes
    const int64_t at = (int64_t)(id - t.first[i]) * CHUNK;
    const int64_t left = t.n[i] - at;
    if (t.in_type[i] == PT_CLIP_F32) {
      chunk_scale((const float*)t.in[i] + at, (float*)t.out[i] + at, left, k);
    } else if (t.in_type[i] == PT_CLIP_BF16) {
      if (t.out_type[i] == PT_CLIP_F32) chunk_scale((const __bf16*)t.in[i] + at, (float*)t.out[i] + at, left, k);
      else chunk_scale((const __bf16*)t.in[i] + at, (__bf16*)t.out[i] + at, left, k);
    } else {
      if (t.out_type[i] == PT_CLIP_F32) chunk_scale((const _Float16*)t.in[i] + at, (float*)t.out[i] + at, left, k);
      else chunk_scale((const _Float16*)t.in[i] + at, (_Float16*)t.out[i] + at, left, k);
    }
  }
}

// ------------------------------------------------------------------ host

int size_of(int type) { return type == PT_CLIP_F32 ? 4 : 2; }

// The next launch's tensors, from t[at]: fills `tab`, returns where the one after starts.
int64_t next_table(const pt_clip_tensor* t, int64_t count, int64_t at, Table& tab) {
  tab.count = 0;
  uint64_t chunks = 0;
  for (; at < count && tab.count < TABLE; ++at) {
    if (t[at].n == 0) continue;
    const uint64_t c = (uint64_t)((t[at].n + CHUNK - 1) / CHUNK);
    if (chunks + c > 0xfff00000u) break;                 // (the grid's stride may not wrap)
    const int k = tab.count++;
    tab.in[k] = t[at].grad;
    tab.out[k] = t[at].out;
    tab.n[k] = t[at].n;
    tab.in_type[k] = (uint8_t)t[at].grad_type;
    tab.out_type[k] = (uint8_t)t[at].out_type;
    tab.first[k] = (uint32_t)chunks;
    chunks += c;
  }
  tab.first[tab.count] = (uint32_t)chunks;
  return at;
}

unsigned grid_of(const Table& tab) {
  return std::min<uint32_t>(tab.first[tab.count], GRID);
}

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
  Table tab;
  int64_t parts = 0, at = 0;
  while (at < count) {
    at = next_table(t, count, at, tab);
    parts += grid_of(tab);
  }
  return parts;
}

template <int P>
int run(const pt_clip_tensor* t, int64_t count, bool scale, double max_norm, float* norm, double* part,
        hipStream_t s) {
  Table tab;
  int64_t parts = 0;
  std::vector<int64_t> starts;
  for (int64_t at = 0; at < count;) {
    starts.push_back(at);
    at = next_table(t, count, at, tab);
    const unsigned g = grid_of(tab);
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
  if (scale)
    for (size_t k = starts.size(); k-- > 0;) {
      next_table(t, count, starts[k], tab);
      const unsigned g = grid_of(tab);
      if (!g) continue;
      hipLaunchKernelGGL((k_scale<P>), dim3(g), dim3(NT), 0, s, tab, from, n, max_norm, norm);
      norm = nullptr;
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
