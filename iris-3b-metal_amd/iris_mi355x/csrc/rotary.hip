// Rotary positions of query, key (and passed-through value) heads: half and interleaved pair layouts,
// part of a head or all of it, any frequencies.
//
// Pair i < pairs of a head at position p turns by the angle a = p f_i:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,  c = t cos a, s = t sin a (t the attention factor of a scaled
//   context), with (x0, x1) = elements (i, i + pairs) (half) or (2 i, 2 i + 1) (interleaved); elements
//   from 2 pairs on are copied. The gradient with regard to x is the transposed rotation, s -> -s.
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there: at position 2^20 an FP32
// product is already 0.06 radians off. cos and sin of the reduced turn are FP32, the rotation FP32 with
// one rounding to the output type.
#include "iris_common.hpp"

namespace iris {
namespace {

constexpr int kMaxTensors = 3;
constexpr int kTurn = 1, kToRows = 2;  // flags: rotate the heads; write to the rows of `rows`

struct RotaryTensor {
  const void* x;
  void* out;
  long xs_b, xs_n, xs_h;  // strides in elements: batch, token, head
  long os_b, os_h, os_n;  // batch, head, row
  long out_rows;
  int heads, flags;
};
struct RotaryArgs {
  RotaryTensor t[kMaxTensors];
  int tensors, heads_total;
  long tokens;
  int head_dim, pairs, interleaved;
  const void* positions;
  const void* rows;
  int positions64, rows64;
  long positions_stride, rows_stride;
  const double* freqs;
  float factor, sign;
};

__device__ __forceinline__ long index_at(const void* p, int wide, long i) {
  return wide ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// (cos, sin)(p f) in FP32 from the 64-bit angle.
__device__ __forceinline__ void turn_of(double p, double f, float& c, float& s) {
  double turn = p * f * 0.15915494309189533576888;  // 1 / (2 pi)
  turn -= rint(turn);
  sincospif(static_cast<float>(2.0 * turn), &s, &c);
}

// One workgroup per (token, batch item); a thread per pair (or pair of copied elements).
template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const long n = blockIdx.x;
  const int b = blockIdx.y;
  const double p = static_cast<double>(index_at(a.positions, a.positions64, b * a.positions_stride + n));
  const int half = a.head_dim / 2;
  for (int i = threadIdx.x; i < a.heads_total * half; i += blockDim.x) {
    int h = i / half;
    const int pair = i - h * half;
    int j = 0;
    while (h >= a.t[j].heads) h -= a.t[j++].heads;
    const RotaryTensor& t = a.t[j];
    const long row = (t.flags & kToRows) ? index_at(a.rows, a.rows64, b * a.rows_stride + n) : n;
    if (row < 0 || row >= t.out_rows) continue;
    const bool turned = (t.flags & kTurn) && pair < a.pairs;
    const int e0 = turned && !a.interleaved ? pair : 2 * pair;
    const int e1 = turned && !a.interleaved ? pair + a.pairs : 2 * pair + 1;
    const T* x = static_cast<const T*>(t.x) + b * t.xs_b + n * t.xs_n + h * t.xs_h;
    T* y = static_cast<T*>(t.out) + b * t.os_b + h * t.os_h + row * t.os_n;
    const T x0 = x[e0], x1 = x[e1];
    if (!turned) {
      y[e0] = x0;
      y[e1] = x1;
      continue;
    }
    float c, s;
    turn_of(p, a.freqs[pair], c, s);
    c *= a.factor;
    s *= a.factor * a.sign;
    const float f0 = to_f32(x0), f1 = to_f32(x1);
    y[e0] = from_f32<T>(__builtin_fmaf(f0, c, -(f1 * s)));
    y[e1] = from_f32<T>(__builtin_fmaf(f1, c, f0 * s));
  }
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_rotary(int tensors, const void* const* x, const long* x_strides, void* const* out,
                           const long* out_strides, const int* heads, const int* flags, const long* out_rows,
                           int dtype, int batch, long tokens, int head_dim, const void* positions,
                           int positions_kind, long positions_stride, const void* rows, int rows_kind,
                           long rows_stride, const double* freqs, int pairs, int layout, float factor, int transpose,
                           hipStream_t stream) {
  IRIS_REQUIRE(tensors >= 1 && tensors <= kMaxTensors && x && x_strides && out && out_strides && heads && flags &&
                   out_rows,
               "rotary: takes one to three tensors");
  IRIS_REQUIRE(dtype == IRIS_F32 || dtype == IRIS_BF16, "rotary: unknown dtype %d", dtype);
  IRIS_REQUIRE(batch >= 0 && batch < 65536 && tokens >= 0 && tokens < (1L << 31), "rotary: bad batch or token count");
  IRIS_REQUIRE(head_dim > 0 && head_dim % 2 == 0 && head_dim <= 1024 && pairs > 0 && 2 * pairs <= head_dim,
               "rotary: need an even head width up to 1024 that holds the %d rotated pairs (got %d)", pairs, head_dim);
  IRIS_REQUIRE(layout == IRIS_ROTARY_HALF || layout == IRIS_ROTARY_INTERLEAVED, "rotary: unknown layout %d", layout);
  if (batch == 0 || tokens == 0) return IRIS_OK;
  IRIS_REQUIRE(positions && freqs, "rotary: null pointer");
  IRIS_REQUIRE(positions_kind == 1 || positions_kind == 3, "rotary: positions are int32 (1) or int64 (3)");
  RotaryArgs a{};
  for (int i = 0; i < tensors; ++i) {
    IRIS_REQUIRE(x[i] && out[i] && heads[i] > 0 && out_rows[i] >= 0, "rotary: tensor %d: null pointer or bad sizes", i);
    IRIS_REQUIRE(!(flags[i] & kToRows) || (rows && (rows_kind == 1 || rows_kind == 3)),
                 "rotary: tensor %d goes to rows, which are missing or neither int32 (1) nor int64 (3)", i);
    IRIS_REQUIRE((flags[i] & kToRows) || out_rows[i] >= tokens, "rotary: output %d holds fewer rows than tokens", i);
    a.t[i] = RotaryTensor{x[i],
                          out[i],
                          x_strides[3 * i],
                          x_strides[3 * i + 1],
                          x_strides[3 * i + 2],
                          out_strides[3 * i],
                          out_strides[3 * i + 1],
                          out_strides[3 * i + 2],
                          out_rows[i],
                          heads[i],
                          flags[i]};
    a.heads_total += heads[i];
  }
  IRIS_REQUIRE(a.heads_total <= 65536, "rotary: too many heads");
  a.tensors = tensors;
  a.tokens = tokens;
  a.head_dim = head_dim;
  a.pairs = pairs;
  a.interleaved = layout == IRIS_ROTARY_INTERLEAVED;
  a.positions = positions;
  a.positions64 = positions_kind == 3;
  a.positions_stride = positions_stride;
  a.rows = rows;
  a.rows64 = rows_kind == 3;
  a.rows_stride = rows_stride;
  a.freqs = freqs;
  a.factor = factor;
  a.sign = transpose ? -1.0f : 1.0f;
  const dim3 grid(static_cast<unsigned>(tokens), batch);
  if (dtype == IRIS_F32)
    rotary_kernel<float><<<grid, 256, 0, stream>>>(a);
  else
    rotary_kernel<bf16><<<grid, 256, 0, stream>>>(a);
  return check_launch("rotary");
}
