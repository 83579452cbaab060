// Attention with a sliding window and a few first tokens that stay visible, 128-wide heads with grouped
// K/V heads: whole prompts, and one or a few queries over a long cache.
//
// Query t of batch item b stands at position p = start[b] + t. Key j < length[b] is visible to it iff
//   (no causal limit or j <= p) and (no window or |p - j| < window or j < sinks) and key_mask[b, j] != 0,
// so a query's keys are [0, sink_end) and [low, high) less the masked ones (Span). The result is
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m) over its visible keys (m their largest
//   score), and 0 where nothing is visible.
#include "iris_common.hpp"

namespace iris {
namespace {

constexpr int kHd = 128;

struct WindowArgs {
  const bf16 *q, *k, *v;
  bf16* out;
  long qs_b, qs_h, qs_n, ks_b, ks_h, ks_n, vs_b, vs_h, vs_n, os_b, os_n;  // strides in elements
  int batch, heads, kv_heads, n_q, n_k;
  long window, sinks;  // window 0: none
  int causal;
  const void *lengths, *starts;
  int lengths64, starts_kind;  // starts_kind 0: length - n_q, 1 int32, 3 int64, 4: `start`
  long start;
  const unsigned char* key_mask;
  long mask_stride;
  float scale_log2;
};

__host__ __device__ __forceinline__ long clamp_long(long x, long lo, long hi) { return x < lo ? lo : (x > hi ? hi : x); }

// Keys of item b that exist, and the position of its first query.
__device__ __forceinline__ int item_length(const WindowArgs& p, int b) {
  if (!p.lengths) return p.n_k;
  const long n = p.lengths64 ? static_cast<const long long*>(p.lengths)[b] : static_cast<const int*>(p.lengths)[b];
  return static_cast<int>(clamp_long(n, 0, p.n_k));
}
__device__ __forceinline__ long item_start(const WindowArgs& p, int b, int length) {
  if (p.starts_kind == 0) return static_cast<long>(length) - p.n_q;
  const long s = p.starts_kind == 4   ? p.start
                 : p.starts_kind == 3 ? static_cast<long>(static_cast<const long long*>(p.starts)[b])
                                      : static_cast<const int*>(p.starts)[b];
  return clamp_long(s, -(1L << 60), 1L << 60);
}

// Visible keys of a query at `pos`: [0, sink_end) and [low, high), low >= sink_end where both hold keys.
struct Span {
  int sink_end, low, high;
};
__device__ __forceinline__ Span span_of(const WindowArgs& p, long pos, int length) {
  Span s;
  s.high = static_cast<int>(p.causal ? clamp_long(pos + 1, 0, length) : p.window ? clamp_long(pos + p.window, 0, length) : length);
  s.low = p.window ? static_cast<int>(clamp_long(pos - p.window + 1, 0, p.n_k)) : 0;
  s.sink_end = p.window ? static_cast<int>(clamp_long(p.causal && pos + 1 < p.sinks ? pos + 1 : p.sinks, 0, length)) : 0;
  if (s.low < s.sink_end) s.low = s.sink_end;
  return s;
}

// One wave per (item, head, query): lane l holds dims 2 l and 2 l + 1, one key at a time.
__global__ __launch_bounds__(256) void window_rows_kernel(WindowArgs p, long total) {
  const long id = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (id >= total) return;
  const int lane = threadIdx.x & 63;
  const int t = static_cast<int>(id % p.n_q);
  const int h = static_cast<int>(id / p.n_q % p.heads);
  const int b = static_cast<int>(id / p.n_q / p.heads);
  const int hk = h / (p.heads / p.kv_heads);
  const bf16* q = p.q + b * p.qs_b + h * p.qs_h + t * p.qs_n + 2 * lane;
  const bf16* k = p.k + b * p.ks_b + hk * p.ks_h + 2 * lane;
  const bf16* v = p.v + b * p.vs_b + hk * p.vs_h + 2 * lane;
  const unsigned char* mask = p.key_mask ? p.key_mask + b * p.mask_stride : nullptr;
  const int length = item_length(p, b);
  const Span s = span_of(p, item_start(p, b, length) + t, length);
  const float q0 = to_f32(q[0]), q1 = to_f32(q[1]);
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  auto key = [&](long j) {
    if (mask && !mask[j]) return;
    const bf16x2 kk = *reinterpret_cast<const bf16x2*>(k + j * p.ks_n);
    const bf16x2 vv = *reinterpret_cast<const bf16x2*>(v + j * p.vs_n);
    const float x = wave_sum(q0 * to_f32(kk[0]) + q1 * to_f32(kk[1])) * p.scale_log2;
    const float top = fmaxf(m, x);
    const float a = top == m ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    const float e = __builtin_amdgcn_exp2f(x - top);
    m = top;
    l = l * a + e;
    o0 = o0 * a + e * to_f32(vv[0]);
    o1 = o1 * a + e * to_f32(vv[1]);
  };
  for (int j = 0; j < s.sink_end; ++j) key(j);
  for (int j = s.low; j < s.high; ++j) key(j);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  bf16* out = p.out + b * p.os_b + t * p.os_n + h * kHd + 2 * lane;
  *reinterpret_cast<bf16x2*>(out) = bf16x2{from_f32<bf16>(o0 * inv), from_f32<bf16>(o1 * inv)};
}

}  // namespace
}  // namespace iris

using namespace iris;

namespace {
void extent(const void* p, const long* shape, const long* strides, int dims, uintptr_t* lo, uintptr_t* hi) {
  long first = 0, last = 0;
  for (int i = 0; i < dims; ++i) (strides[i] < 0 ? first : last) += (shape[i] - 1) * strides[i];
  *lo = reinterpret_cast<uintptr_t>(p) + first * 2;
  *hi = reinterpret_cast<uintptr_t>(p) + (last + 1) * 2;
}

// Checks the arguments and turns them into the kernels' form; p.batch stays 0 where there is nothing to do.
int window_args(const iris_window_attn_args* args, WindowArgs& p) {
  IRIS_REQUIRE(args, "window_attn: null pointer");
  const iris_window_attn_args& g = *args;
  const long batch = g.q_shape[0], heads = g.q_shape[1], n_q = g.q_shape[2], kv_heads = g.k_shape[1], n_k = g.k_shape[2];
  for (int i = 0; i < 4; ++i)
    IRIS_REQUIRE(g.k_shape[i] == g.v_shape[i], "window_attn: k and v must be of one shape");
  IRIS_REQUIRE(batch >= 0 && batch < 65536 && heads > 0 && kv_heads > 0 && heads <= 65536 && heads % kv_heads == 0 &&
                   g.k_shape[0] == batch && g.q_shape[3] == kHd && g.k_shape[3] == kHd,
               "window_attn: q [%ld, %ld, %ld, %ld] and k / v [%ld, %ld, %ld, %ld] do not match: one batch, 128-wide heads, "
               "a multiple of K/V heads",
               batch, heads, n_q, g.q_shape[3], g.k_shape[0], kv_heads, n_k, g.k_shape[3]);
  IRIS_REQUIRE(n_q >= 0 && n_k >= 0 && n_q < (1L << 30) && n_k < (1L << 30), "window_attn: need fewer than 2^30 rows");
  IRIS_REQUIRE(g.window >= 0 && g.sinks >= 0, "window_attn: window and sinks must not be negative");
  IRIS_REQUIRE(!g.lengths || g.lengths_kind == 1 || g.lengths_kind == 3, "window_attn: lengths are int32 (1) or int64 (3)");
  IRIS_REQUIRE(g.starts_kind == 0 || g.starts_kind == 4 || ((g.starts_kind == 1 || g.starts_kind == 3) && g.starts),
               "window_attn: starts are int32 (1), int64 (3), one value (4) or absent (0)");
  IRIS_REQUIRE(g.out_shape[0] == batch && g.out_shape[1] == n_q && g.out_shape[2] == heads * kHd && g.out_strides[2] == 1,
               "window_attn: out must be [%ld, %ld, %ld] with unit column stride", batch, n_q, heads * kHd);
  IRIS_REQUIRE(g.q_strides[3] == 1 && g.k_strides[3] == 1 && g.v_strides[3] == 1,
               "window_attn: heads must have unit stride");
  if (batch == 0 || n_q == 0) return IRIS_OK;
  IRIS_REQUIRE(g.q && g.out && (n_k == 0 || (g.k && g.v)), "window_attn: null pointer");
  IRIS_REQUIRE(aligned(g.q, 16) && aligned(g.k, 16) && aligned(g.v, 16) && aligned(g.out, 8),
               "window_attn: inputs must be 16-byte aligned, the output 8");
  for (int i = 0; i < 3; ++i)
    IRIS_REQUIRE(g.q_strides[i] % 8 == 0 && g.k_strides[i] % 8 == 0 && g.v_strides[i] % 8 == 0,
                 "window_attn: strides must be multiples of 8 elements");
  IRIS_REQUIRE((n_q == 1 || g.out_strides[1] >= heads * kHd) && (batch == 1 || g.out_strides[0] >= heads * kHd) &&
                   g.out_strides[0] % 4 == 0 && g.out_strides[1] % 4 == 0,
               "window_attn: output rows must not overlap, strides must be multiples of 4");
  uintptr_t o0, o1, x0, x1;
  extent(g.out, g.out_shape, g.out_strides, 3, &o0, &o1);
  const void* in[3] = {g.q, g.k, g.v};
  const long* shapes[3] = {g.q_shape, g.k_shape, g.v_shape};
  const long* strides[3] = {g.q_strides, g.k_strides, g.v_strides};
  for (int i = 0; i < (n_k ? 3 : 1); ++i) {
    extent(in[i], shapes[i], strides[i], 4, &x0, &x1);
    IRIS_REQUIRE(o1 <= x0 || x1 <= o0, "window_attn: out must lie apart from q, k and v");
  }
  p.q = static_cast<const bf16*>(g.q);
  p.k = static_cast<const bf16*>(g.k);
  p.v = static_cast<const bf16*>(g.v);
  p.out = static_cast<bf16*>(g.out);
  p.qs_b = g.q_strides[0], p.qs_h = g.q_strides[1], p.qs_n = g.q_strides[2];
  p.ks_b = g.k_strides[0], p.ks_h = g.k_strides[1], p.ks_n = g.k_strides[2];
  p.vs_b = g.v_strides[0], p.vs_h = g.v_strides[1], p.vs_n = g.v_strides[2];
  p.os_b = g.out_strides[0], p.os_n = g.out_strides[1];
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.n_q = static_cast<int>(n_q);
  p.n_k = static_cast<int>(n_k);
  p.window = g.window < (1L << 60) ? g.window : (1L << 60);
  p.sinks = g.sinks;
  p.causal = g.causal != 0;
  p.lengths = g.lengths;
  p.lengths64 = g.lengths_kind == 3;
  p.starts = g.starts;
  p.starts_kind = static_cast<int>(g.starts_kind);
  p.start = clamp_long(g.start, -(1L << 60), 1L << 60);
  p.key_mask = static_cast<const unsigned char*>(g.key_mask);
  p.mask_stride = g.mask_stride;
  p.scale_log2 = static_cast<float>(g.scale * 1.4426950408889634);
  return IRIS_OK;
}
}  // namespace

extern "C" int iris_window_attn_workspace(const iris_window_attn_args* args, long* bytes) {
  IRIS_REQUIRE(args && bytes, "window_attn: null pointer");
  *bytes = 0;
  return IRIS_OK;
}

extern "C" int iris_window_attn(const iris_window_attn_args* args, hipStream_t stream) {
  WindowArgs p{};
  const int rc = window_args(args, p);
  if (rc || p.batch == 0) return rc;
  const long total = static_cast<long>(p.batch) * p.heads * p.n_q;
  IRIS_REQUIRE(total < (1L << 31), "window_attn: grid too large");
  window_rows_kernel<<<dim3(static_cast<unsigned>((total + 3) / 4)), 256, 0, stream>>>(p, total);
  return check_launch("window_attn");
}
