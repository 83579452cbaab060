// Rotary positions of query, key (and passed-through value) heads: half and interleaved pair layouts,
// part of a head or all of it, any frequencies.
//
// Pair i < pairs of a head at position p turns by the angle a = p f_i:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,  c = t cos a, s = t sin a (t the attention factor of a scaled
//   context), with (x0, x1) = elements (i, i + pairs) (half) or (2 i, 2 i + 1) (interleaved); elements
//   from 2 pairs on are copied. The gradient with regard to x is the transposed rotation, s -> -s.
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there: at position 2^20 an FP32
// product is already 0.06 radians off. cos and sin of the reduced turn, rounded to FP32 (2^-22 of a radian at
// worst), are FP32, the rotation FP32 with one rounding to the output type: FP32 heads end 5.0e-8 from 64 bits
// in norm where 64-bit cos and sin leave 4.2e-8.
//
// Bound by memory: every element is read and written once. A workgroup takes `tok` tokens of one item and
// tensor, computes their (cos, sin) into LDS once for all heads, and moves the heads in chunks of 16 bytes
// (both halves of a pair chunk in one thread, so that a rotation in place is safe); consecutive threads take
// consecutive chunks of a head, then the next head of the token; a thread's loads of four heads go out
// together, the first before the angles. Odd widths and strides, and unaligned tensors, go element by element
// through the same code. 4.4 TB/s at 32768 tokens of 32 + 8 BF16 heads (a copy of that size class moves 4.9),
// 3.2 us for one token of 20 + 5 + 5 heads, 5.1 TB/s at 2 x 4097 FP32 tokens (partly from the cache); element by
// element 2.0 TB/s (32768 tokens of 40 BF16 heads of 80, 20 turned: 209 us; 40 turned 168, 80 turned 107).
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
  // items of a head: rotated ones (two chunks in the half layout, one in the interleaved), then copied chunks; threads
  // per head, heads side by side, and the tokens and heads from a thread's head to its next
  int turning, items, lanes, slots, step_tok, step_h;
};
struct RotaryArgs {
  RotaryTensor t[kMaxTensors];
  int tensors;
  long tokens;
  int tok;  // tokens per workgroup
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

template <typename T, int N>
struct Chunk {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Chunk<T, N> load_chunk(const T* p) {
  Chunk<T, N> c;
  if constexpr (N * sizeof(T) == 16) {
    *reinterpret_cast<int4*>(&c) = *reinterpret_cast<const int4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) c.v[i] = p[i];
  }
  return c;
}
template <typename T, int N>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T, N>& c) {
  if constexpr (N * sizeof(T) == 16) {
    *reinterpret_cast<int4*>(p) = *reinterpret_cast<const int4*>(&c);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = c.v[i];
  }
}

// VEC: elements per chunk (16 bytes, or 1: half layout, 2: interleaved, by single elements).
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  extern __shared__ f32x2 turns[];  // [tok][pairs] (cos, sin)
  constexpr int U = 4;              // heads of a thread whose loads are underway together
  const long n0 = static_cast<long>(blockIdx.x) * a.tok;
  const int b = blockIdx.y;
  const RotaryTensor& t = a.t[blockIdx.z];
  const int turned = (t.flags & kTurn) ? a.pairs : 0;
  const bool to_rows = t.flags & kToRows;
  const int ntok = static_cast<int>(a.tokens - n0 < a.tok ? a.tokens - n0 : a.tok);
  bool ready = false;  // the first loads go out before the angles are computed
  auto angles = [&]() {
    if (ready || turned == 0) return;
    ready = true;
    for (int i = threadIdx.x; i < ntok * a.pairs; i += 256) {
      const int t = i / a.pairs, pair = i - t * a.pairs;
      const double p = static_cast<double>(index_at(a.positions, a.positions64, b * a.positions_stride + n0 + t));
      float c, s;
      turn_of(p, a.freqs[pair], c, s);
      turns[i] = f32x2{c * a.factor, s * a.factor * a.sign};
    }
    __syncthreads();
  };
  const int heads = t.heads, turning = t.turning, items = t.items, lanes = t.lanes;
  const int slot = static_cast<int>(threadIdx.x) / lanes, c0 = threadIdx.x - slot * lanes;
  const bool on = slot < t.slots;
  const long x_step = t.step_tok * t.xs_n + t.step_h * t.xs_h, y_step = t.step_h * t.os_h;
  const long x_wrap = t.xs_n - heads * t.xs_h, y_wrap = heads * t.os_h;
  const T* const x0 = static_cast<const T*>(t.x) + b * t.xs_b + n0 * t.xs_n;
  T* const y0 = static_cast<T*>(t.out) + b * t.os_b;
  for (int c = c0; c - c0 < items; c += lanes) {
    const bool half = !INTERLEAVED && c < turning;
    const bool copy = c >= turning;
    const int e = copy ? 2 * turned + (c - turning) * VEC : c * VEC;
    const bool here = on && c < items;
    // (the thread's next head and the offsets of its token and head, kept up by additions)
    int tok = slot / heads, h = slot - tok * heads;
    long xo = tok * t.xs_n + h * t.xs_h, yo = h * t.os_h;
    while (true) {
      Chunk<T, VEC> u[U], v[U];
      int toks[U];
      long ys[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        toks[i] = here && tok < ntok ? tok : -1;
        ys[i] = yo;
        if (toks[i] >= 0) {
          u[i] = load_chunk<T, VEC>(x0 + xo + e);
          if (half) v[i] = load_chunk<T, VEC>(x0 + xo + e + turned);
        }
        tok += t.step_tok, h += t.step_h, xo += x_step, yo += y_step;
        if (h >= heads) h -= heads, ++tok, xo += x_wrap, yo -= y_wrap;
      }
      angles();
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (toks[i] < 0) continue;
        const long n = n0 + toks[i];
        const long row = to_rows ? index_at(a.rows, a.rows64, b * a.rows_stride + n) : n;
        if (row < 0 || row >= t.out_rows) continue;
        T* const y = y0 + ys[i] + row * t.os_n + e;
        const f32x2* cs = turns + toks[i] * a.pairs + (INTERLEAVED ? e / 2 : e);
        if (copy) {
        } else if constexpr (INTERLEAVED) {
#pragma unroll
          for (int q = 0; q < VEC / 2; ++q) {
            const float f0 = to_f32(u[i].v[2 * q]), f1 = to_f32(u[i].v[2 * q + 1]);
            const f32x2 r = cs[q];
            u[i].v[2 * q] = from_f32<T>(__builtin_fmaf(f0, r[0], -(f1 * r[1])));
            u[i].v[2 * q + 1] = from_f32<T>(__builtin_fmaf(f1, r[0], f0 * r[1]));
          }
        } else {
#pragma unroll
          for (int q = 0; q < VEC; ++q) {
            const float f0 = to_f32(u[i].v[q]), f1 = to_f32(v[i].v[q]);
            const f32x2 r = cs[q];
            u[i].v[q] = from_f32<T>(__builtin_fmaf(f0, r[0], -(f1 * r[1])));
            v[i].v[q] = from_f32<T>(__builtin_fmaf(f1, r[0], f0 * r[1]));
          }
          store_chunk<T, VEC>(y + turned, v[i]);
        }
        store_chunk<T, VEC>(y, u[i]);
      }
      if (tok >= ntok) break;
    }
  }
}

template <typename T>
void launch_rotary(const RotaryArgs& a, bool vector, int batch, hipStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  const dim3 grid(static_cast<unsigned>((a.tokens + a.tok - 1) / a.tok), batch, a.tensors);
  const size_t lds = static_cast<size_t>(a.tok) * a.pairs * sizeof(f32x2);
  if (a.interleaved) {
    if (vector)
      rotary_kernel<T, kVec, true><<<grid, 256, lds, stream>>>(a);
    else
      rotary_kernel<T, 2, true><<<grid, 256, lds, stream>>>(a);
  } else {
    if (vector)
      rotary_kernel<T, kVec, false><<<grid, 256, lds, stream>>>(a);
    else
      rotary_kernel<T, 1, false><<<grid, 256, lds, stream>>>(a);
  }
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_rotary(const iris_rotary_args* args, hipStream_t stream) {
  IRIS_REQUIRE(args, "rotary: null pointer");
  const iris_rotary_args& g = *args;
  IRIS_REQUIRE(g.tensors >= 1 && g.tensors <= kMaxTensors && g.turned >= 0 && g.to_rows >= 0,
               "rotary: takes one to three tensors");
  IRIS_REQUIRE(g.dtype == IRIS_F32 || g.dtype == IRIS_BF16, "rotary: unknown dtype %ld", g.dtype);
  const long batch = g.t[0].x_shape[0], tokens = g.t[0].x_shape[1], dim = g.t[0].x_shape[3];
  IRIS_REQUIRE(batch >= 0 && batch < 65536 && tokens >= 0 && tokens < (1L << 31), "rotary: bad batch or token count");
  IRIS_REQUIRE(dim > 0 && dim % 2 == 0 && dim <= 1024 && g.pairs > 0 && 2 * g.pairs <= dim,
               "rotary: need an even head width up to 1024 that holds the %ld rotated pairs (got %ld)", g.pairs, dim);
  IRIS_REQUIRE(g.layout == IRIS_ROTARY_HALF || g.layout == IRIS_ROTARY_INTERLEAVED, "rotary: unknown layout %ld", g.layout);
  IRIS_REQUIRE(g.positions_kind == 1 || g.positions_kind == 3, "rotary: positions are int32 (1) or int64 (3)");
  const int size = g.dtype == IRIS_F32 ? 4 : 2;
  RotaryArgs a{};
  StridedRuns xs[kMaxTensors] = {}, outs[kMaxTensors] = {};
  for (int i = 0; i < g.tensors; ++i) {
    const iris_rotary_tensor& t = g.t[i];
    const long heads = t.x_shape[2], rows = t.out_shape[2];
    const bool to_rows = i >= g.to_rows;
    IRIS_REQUIRE(t.x_shape[0] == batch && t.x_shape[1] == tokens && t.x_shape[3] == dim && heads > 0 && heads <= 4096 &&
                     t.x_strides[3] == 1,
                 "rotary: tensor %d: heads must be [%ld, %ld, H, %ld] with unit stride in a head", i, batch, tokens, dim);
    IRIS_REQUIRE(t.out_shape[0] == batch && t.out_shape[1] == heads && t.out_shape[3] == dim && rows >= 0 &&
                     rows < (1L << 40) && (to_rows || rows == tokens) && t.out_strides[3] == 1,
                 "rotary: output %d must be [%ld, %ld, %s, %ld] with unit stride in a head", i, batch, heads,
                 to_rows ? "rows" : "tokens", dim);
    IRIS_REQUIRE(!to_rows || g.rows_kind == 1 || g.rows_kind == 3, "rotary: rows are int32 (1) or int64 (3)");
    a.t[i] = RotaryTensor{t.x,
                          t.out,
                          t.x_strides[0],
                          t.x_strides[1],
                          t.x_strides[2],
                          t.out_strides[0],
                          t.out_strides[1],
                          t.out_strides[2],
                          rows,
                          static_cast<int>(heads),
                          (i < g.turned ? kTurn : 0) | (to_rows ? kToRows : 0)};
    if (batch == 0 || tokens == 0) continue;
    IRIS_REQUIRE(t.x && (t.out || rows == 0) && g.positions && g.freqs && (!to_rows || g.rows), "rotary: null pointer");
    if (rows == 0) continue;  // (read all the same, and dropped)
    xs[i] = strided_runs(t.x, t.x_shape, t.x_strides, 3, size, dim);
    outs[i] = strided_runs(t.out, t.out_shape, t.out_strides, 3, size, dim);
    IRIS_REQUIRE(!share_memory(outs[i], outs[i]), "rotary: output %d is an expanded tensor, or its heads overlap", i);
    const bool same = t.x == t.out && !to_rows && (batch == 1 || t.x_strides[0] == t.out_strides[0]) &&
                      (tokens == 1 || t.x_strides[1] == t.out_strides[2]) &&
                      (heads == 1 || t.x_strides[2] == t.out_strides[1]);
    IRIS_REQUIRE(same || !share_memory(xs[i], outs[i]),
                 "rotary: output %d must be its input itself (as [B, H, N, D]) or lie apart from it", i);
  }
  if (batch == 0 || tokens == 0) return IRIS_OK;
  // (tensors of one projection interleave: their extents meet, their heads do not)
  for (int i = 0; i < g.tensors; ++i)
    for (int j = 0; j < g.tensors; ++j)
      IRIS_REQUIRE(i == j || !outs[i].p || !outs[j].p ||
                       (!share_memory(outs[i], xs[j]) && (j < i || !share_memory(outs[i], outs[j]))),
                   "rotary: output %d shares memory with another tensor's input or output", i);
  a.tensors = static_cast<int>(g.tensors);
  a.tokens = tokens;
  a.head_dim = static_cast<int>(dim);
  a.pairs = static_cast<int>(g.pairs);
  a.interleaved = g.layout == IRIS_ROTARY_INTERLEAVED;
  a.positions = g.positions;
  a.positions64 = g.positions_kind == 3;
  a.positions_stride = g.positions_stride;
  a.rows = g.rows;
  a.rows64 = g.rows_kind == 3;
  a.rows_stride = g.rows_stride;
  a.freqs = g.freqs;
  a.factor = static_cast<float>(g.factor);
  a.sign = g.transpose ? -1.0f : 1.0f;
  // tokens per workgroup, up to eight: four workgroups for every CU (us of 4 x 300 tokens, 20 / 5 heads, at 2, 4, 8 for
  // every CU: 9.3 / 7.7 / 12.0; 2000 tokens, 32 / 8 heads: 13.3 / 12.2 / 14.2; larger calls alike)
  const long per = batch * tokens * g.tensors / (4 * device_cus());
  a.tok = static_cast<int>(per < 1 ? 1 : (per > 8 ? 8 : per));
  IRIS_REQUIRE((tokens + a.tok - 1) / a.tok < (1L << 24), "rotary: too many tokens");
  // chunks of 16 bytes where every chunk of every head is aligned and whole
  const long vec = 16 / size;
  bool vector = (a.interleaved ? 2 * g.pairs : g.pairs) % vec == 0 && (dim - 2 * g.pairs) % vec == 0;
  for (int i = 0; i < g.tensors; ++i) {
    const iris_rotary_tensor& t = g.t[i];
    vector = vector && aligned(t.x, 16) && aligned(t.out, 16);
    for (int d = 0; d < 3; ++d) vector = vector && t.x_strides[d] % vec == 0 && t.out_strides[d] % vec == 0;
  }
  for (int i = 0; i < g.tensors; ++i) {
    RotaryTensor& t = a.t[i];
    const int turned = (t.flags & kTurn) ? a.pairs : 0;
    const int chunk = vector ? static_cast<int>(vec) : a.interleaved ? 2 : 1;
    t.turning = (a.interleaved ? 2 * turned : turned) / chunk;
    t.items = t.turning + (a.head_dim - 2 * turned) / chunk;
    t.lanes = t.items < 256 ? t.items : 256;
    t.slots = 256 / t.lanes;
    t.step_tok = t.slots / t.heads;
    t.step_h = t.slots % t.heads;
  }
  if (g.dtype == IRIS_F32)
    launch_rotary<float>(a, vector, static_cast<int>(batch), stream);
  else
    launch_rotary<bf16>(a, vector, static_cast<int>(batch), stream);
  return check_launch("rotary");
}
