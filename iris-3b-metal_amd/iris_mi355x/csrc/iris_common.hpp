// Shared types, vector helpers and error reporting for the Iris MI355X (gfx950) kernels.
//
// Every kernel in this library works on caller-owned device memory; entry points
// validate their arguments on the host, launch asynchronously on the given
// stream and return IRIS_OK or a negative IRIS_E_* code (message retrievable
// with iris_last_error()).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/iris_hip.h"

namespace iris {

typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWave = 64;

// ---- host-side error state --------------------------------------------------
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int check_launch(const char* what);

#define IRIS_REQUIRE(cond, ...)                      \
  do {                                               \
    if (!(cond)) return ::iris::fail(IRIS_E_INVALID, __VA_ARGS__); \
  } while (0)

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// ---- memory that strided tensors touch -----------------------------------------
// A tensor of runs of `run` contiguous bytes at p + sum_i j_i strides[i], 0 <= j_i < shape[i].
struct StridedRuns {
  const void* p;
  int dims;
  long shape[4], strides[4];  // strides in bytes, of either sign
  long run;
};
inline StridedRuns strided_runs(const void* p, const long* shape, const long* strides, int dims, int size, long run) {
  StridedRuns t{p, dims, {}, {}, run * size};
  for (int i = 0; i < dims; ++i) t.shape[i] = shape[i], t.strides[i] = strides[i] * size;
  return t;
}

// Whether two such tensors share a byte; with a == b, whether two runs of one tensor do. Exact: two runs share a byte
// iff their addresses' difference, a sum of stride times index difference over the axes, lies within a run; searched
// axis by axis from the largest stride down, where the smaller ones leave one or two index differences to try for
// layouts in use. (A layout that leaves more than 2^14 in all counts as sharing.)
inline bool share_memory(const StridedRuns& a, const StridedRuns& b) {
  struct Term {
    __int128 stride, lo, hi;
  } t[8];
  const bool self = &a == &b;
  int n = 0;
  auto axes = [&](const StridedRuns& x, bool minus) {
    for (int i = 0; i < x.dims; ++i) {
      if (x.shape[i] <= 0) return false;
      if (x.shape[i] == 1 || (x.strides[i] == 0 && !self)) continue;
      const __int128 last = x.shape[i] - 1, s = x.strides[i];
      const bool down = (s < 0) != minus;
      int k = n;  // (one term for both tensors' axes of a stride)
      for (int j = 0; j < n && !self; ++j)
        if (t[j].stride == (s < 0 ? -s : s)) k = j;
      if (k == n) t[n++] = Term{s < 0 ? -s : s, 0, 0};
      if (down || self) t[k].lo -= last;
      if (!down || self) t[k].hi += last;
    }
    return true;
  };
  if (!axes(a, true) || (!self && !axes(b, false))) return false;  // (empty)
  for (int i = 1; i < n; ++i)
    for (int j = i; j > 0 && t[j].stride > t[j - 1].stride; --j) {
      const Term x = t[j];
      t[j] = t[j - 1], t[j - 1] = x;
    }
  __int128 least[9] = {}, most[9] = {};  // of the terms from i on
  for (int i = n - 1; i >= 0; --i) least[i] = least[i + 1] + t[i].stride * t[i].lo, most[i] = most[i + 1] + t[i].stride * t[i].hi;
  if (self) {  // (nested axes, without a search)
    int i = 0;
    while (i < n && t[i].stride >= most[i + 1] + a.run) ++i;
    if (i == n) return false;
  }
  int budget = 1 << 14;
  // whether the terms from i on can add up to a value in [lo, hi]; other: an index differs already
  auto search = [&](auto&& again, int i, __int128 lo, __int128 hi, bool other) -> bool {
    if (--budget < 0) return true;
    if (i == n) return lo <= 0 && hi >= 0 && (other || !self);
    if (most[i] < lo || least[i] > hi) return false;
    __int128 from = t[i].lo, to = t[i].hi;
    if (t[i].stride > 0) {
      auto floor_div = [](__int128 x, __int128 y) { return x / y - (x % y < 0); };
      const __int128 f = -floor_div(-(lo - most[i + 1]), t[i].stride), l = floor_div(hi - least[i + 1], t[i].stride);
      from = f > from ? f : from, to = l < to ? l : to;
    }
    for (__int128 d = from; d <= to; ++d)
      if (again(again, i + 1, lo - d * t[i].stride, hi - d * t[i].stride, other || d != 0)) return true;
    return false;
  };
  // run of b at address difference x from a run of a: they meet for -b.run < x < a.run
  const __int128 base = self ? 0 : static_cast<__int128>(reinterpret_cast<intptr_t>(b.p)) - reinterpret_cast<intptr_t>(a.p);
  return search(search, 0, 1 - b.run - base, a.run - 1 - base, false);
}

// Compute units of the current device (launch shapes that place one workgroup per CU).
inline int device_cus() {
  static int cached[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cached[dev] == 0) {
    int cus = 0;
    cached[dev] = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0
                      ? cus
                      : 256;
  }
  return cached[dev];
}

// ---- device helpers ----------------------------------------------------------
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return static_cast<float>(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return static_cast<bf16>(x); }

// 4-element loads / stores returning / taking FP32.
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4 load4(const bf16* p) {
  const bf16x4 v = *reinterpret_cast<const bf16x4*>(p);
  return f32x4{to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3])};
}
__device__ __forceinline__ void store4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, f32x4 v) {
  *reinterpret_cast<bf16x4*>(p) = bf16x4{from_f32<bf16>(v[0]), from_f32<bf16>(v[1]), from_f32<bf16>(v[2]),
                                         from_f32<bf16>(v[3])};
}

// 8-element loads / stores.
__device__ __forceinline__ void load8(const float* p, float* out) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p);
  const f32x4 b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    out[i] = a[i];
    out[4 + i] = b[i];
  }
}
__device__ __forceinline__ void load8(const bf16* p, float* out) {
  const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = to_f32(v[i]);
}
__device__ __forceinline__ void store8(float* p, const float* v) {
  *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(bf16* p, const float* v) {
  bf16x8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = from_f32<bf16>(v[i]);
  *reinterpret_cast<bf16x8*>(p) = o;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Sum over aligned groups of `width` lanes (width a power of two <= 64).
template <int width>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = width / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// Position of token slot i inside its group of 16 in the V^T layout the attention kernel reads:
// the middle two 4-token quads are swapped (0-3, 8-11, 4-7, 12-15), so that the 8 keys one
// MFMA lane needs (4 g .. 4 g + 3 and 8 + 4 g .. 8 + 4 g + 3) are contiguous. An involution.
__device__ __forceinline__ int vt_slot(int i) {
  const int quad = (i >> 2) & 3;
  return (i & ~15) | ((quad == 1 ? 2 : quad == 2 ? 1 : quad) << 2) | (i & 3);
}

// Per-head RMSNorm + rotary embedding of one 128-wide head: y = rope((a / rms) * w), rms over
// the 128 values (+ eps inside the root), pair j = (2 j, 2 j + 1) rotated by (c[j], s[j]) of its
// position. The head is held as 16 chunks of 8 values (chunk s: elements 8 s .. 8 s + 7, rotary
// pairs 4 s .. 4 s + 3); the squares are summed per chunk in element order, and the 16 chunk sums
// combined as an xor butterfly over chunks 8, 4, 2, 1 apart (head_norm_rope: one chunk per lane
// of an aligned 16-lane group, every lane of which must take part; head_sum_tree: the same
// additions in one thread, equal bits).
// (The fused multiply-adds are spelled out: left to contraction, the compiler fused a different
// product of a two-product sum in different callers, one BF16 step apart now and then.)
__device__ __forceinline__ float head_chunk_sq(const float (&a)[8]) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(a[e], a[e], ss);
  return ss;
}
__device__ __forceinline__ float head_sum_tree(const float (&ss)[16]) {
  float v1[8], v2[4], v3[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) v1[i] = ss[i] + ss[i + 8];
#pragma unroll
  for (int i = 0; i < 4; ++i) v2[i] = v1[i] + v1[i + 4];
#pragma unroll
  for (int i = 0; i < 2; ++i) v3[i] = v2[i] + v2[i + 2];
  return v3[0] + v3[1];
}
__device__ __forceinline__ float head_rms_scale(float sum_sq, float eps) { return rsqrtf(sum_sq / 128.0f + eps); }
__device__ __forceinline__ void head_scale_rope(const float (&a)[8], float r, const float (&w)[8], const f32x4& c,
                                                const f32x4& s, float (&y)[8]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float a0 = (a[2 * p] * r) * w[2 * p];
    const float a1 = (a[2 * p + 1] * r) * w[2 * p + 1];
    y[2 * p] = __builtin_fmaf(a0, c[p], -(a1 * s[p]));
    y[2 * p + 1] = __builtin_fmaf(a0, s[p], a1 * c[p]);
  }
}
__device__ __forceinline__ void head_norm_rope(const float (&a)[8], const float (&w)[8], const f32x4& c,
                                               const f32x4& s, float eps, float (&y)[8]) {
  head_scale_rope(a, head_rms_scale(group_sum<16>(head_chunk_sq(a)), eps), w, c, s, y);
}

// x sigmoid(x) and sigmoid(x) with the hardware reciprocal (~1 ulp) in place of an IEEE division,
// which costs about ten instructions per element in the GEMM and attention epilogues.
__device__ __forceinline__ float silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Workgroups are dispatched round-robin over the 8 XCDs (each with its own L2).
// Map the hardware id to a logical id so that consecutive logical ids run on
// the same XCD; neighbouring logical tiles then share operands in one L2.
__device__ __forceinline__ int xcd_remap(int wg, int total) {
  const int xcd = wg & 7;
  const int local = wg >> 3;
  const int base = total >> 3;
  const int rem = total & 7;
  return xcd * base + (xcd < rem ? xcd : rem) + local;
}

// s_waitcnt with only the vector-memory counter constrained (gfx9 encoding).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// A barrier for what passes through LDS, which leaves loads from memory underway.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Raw buffer resources: word 3 of a gfx9-family buffer descriptor (32-bit dwords, no swizzle).
// A buffer load takes one 32-bit VGPR byte offset and an SGPR offset, and reads past the
// resource's size return zeros instead of faulting.
constexpr int kBufferFlags = 0x00020000;

// 16 bytes per lane from a buffer straight into LDS at lds + 16 * lane (lds wave-uniform). (A
// non-template device function: the host compilation pass never instantiates it, which it would
// reject for the LDS address-space cast, and the kernels calling it keep their launch stubs.)
__device__ __forceinline__ void buffer_load_lds16(__amdgpu_buffer_rsrc_t rsrc, bf16* lds, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, voffset, soffset, 0,
                                           0);
}

}  // namespace iris
