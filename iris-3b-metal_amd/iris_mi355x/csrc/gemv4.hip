// Matrix-vector products with 4-bit weights and group scales, for the calls of a few rows that gemv.hip
// serves with BF16 weights.
//
// W[n, k] = scale[n, k / group] (code[n, k] - zero[n, k / group]), codes 0..15 (element k of a row is the
// low half of byte k / 2 where k is even, the high half where it is odd), zero 8 where none are given;
// y[b, n] = act_out(sum_k W[n, k] act_in(x[b, k]) + bias[n]), out[j, b, n] = y[b, n] + extra_bias[j, n].
//
// Bound by the codes' way from memory: half a byte per weight. The products run on v_mfma_f32_16x16x32_bf16
// with the input rows as A and 16 weight rows as B, because one wave of FMAs per weight and row would
// take longer than the read:
// - B: a lane reads 16 bytes (32 codes) of weight row l % 16; two lane swaps among the four groups of 16
//   lanes turn four such dwords into the B operands of four 32-wide k-steps. (16 + code) is a BF16 value
//   whose mantissa holds the code (0x4180 | code << 3), one shift and one and-or per two weights; the
//   offset leaves by a second MFMA of the same A with -(16 + zero) in every place, exact like the first:
//   what is summed is x (16 + code) and x -(16 + zero), at most 5 times the magnitude of the result's terms.
// - A: BF16 rows as they are; FP32 rows (and activated ones) as three BF16 rows that add up to them exactly
//   (8 + 8 + 8 bits of significand, by truncation), so FP32 inputs keep FP32 products at no extra MFMA while
//   three rows per input row fit 16. They lie in LDS with each 8 elements in the order 0 4 1 5 2 6 3 7 that
//   the codes come in.
// - The FP32 sums of a group of at least 32 are scaled and added to the row's FP32 sums.
// A workgroup's four waves take 64 NT weight rows over all of k, or, where that leaves CUs without work, 16 NT
// rows with k dealt to the waves and their sums joined in LDS.
#include "iris_common.hpp"

namespace iris {
namespace {

constexpr int kDepth = 4;         // code loads (16 rows x 128 k each) in flight per wave and weight tile
constexpr int kMaxRows = 48;      // A rows of a workgroup
constexpr int kLdsBytes = 64 << 10;  // inputs and scales of one stage of k: two workgroups per CU

struct W4Job {
  const unsigned char* codes;
  const void* scales;
  const unsigned char* zeros;
  int n;
  const float *bias, *extra;
  int n_extra;
  void* out;
  int wk;  // waves that share a weight tile's k
  int kc;  // k per stage, a multiple of 128 wk
};
struct W4Launch {
  W4Job job[2];
  int blocks0;
  const void* x;
  int x_dtype, out_dtype, scales_dtype;
  int batch, nb;  // input rows in all, and per workgroup (blockIdx.y)
  int parts;      // A rows per input row: 1, or 3 for FP32 and activated inputs
  int k, group, groups, in_act, out_act;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, long i) {
  return dtype == IRIS_F32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const bf16*>(p)[i]);
}
__device__ __forceinline__ unsigned bits_of(float x) { return __builtin_bit_cast(unsigned, x); }
__device__ __forceinline__ float of_bits(unsigned x) { return __builtin_bit_cast(float, x); }

// LDS of a launch: A rows of kc BF16 + 16 bytes (the 16 rows of a fragment read then start in distinct banks),
// and per weight row and group of a stage the scale and the offset's BF16 pair, rows an odd number of pairs apart.
__host__ __device__ __forceinline__ int x_stride(int kc) { return 2 * kc + 16; }
__host__ __device__ __forceinline__ int stage_groups(int kc, int group) { return ((kc + group - 1) / group + 1) | 1; }

// MT tiles of 16 A rows, NT of 16 weight rows per wave; SPG 32-wide k-steps per scale.
template <int MT, int NT, int SPG>
__global__ __launch_bounds__(256) void gemv_w4_kernel(W4Launch a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const bool second = static_cast<int>(blockIdx.x) >= a.blocks0;
  const W4Job& job = second ? a.job[1] : a.job[0];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = 4 / job.wk, wave_n = w % wn, wave_k = w / wn;
  const int n_wg = wn * NT * 16;
  const int n0 = (static_cast<int>(blockIdx.x) - (second ? a.blocks0 : 0)) * n_wg;
  const int b0 = blockIdx.y * a.nb;
  const int nb = min(a.nb, a.batch - b0);
  const int rows = nb * a.parts;
  const int k = a.k, kc = job.kc, n = job.n;
  const int xs = x_stride(kc), gs = stage_groups(kc, a.group);
  uint2* const sc = reinterpret_cast<uint2*>(lds + a.nb * a.parts * xs);  // [n_wg][gs]
  __shared__ unsigned bad;  // input rows (of this workgroup) with a value that is not finite

  const unsigned char* codes[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    codes[t] = job.codes + static_cast<long>(min(n0 + (wave_n * NT + t) * 16 + l16, n - 1)) * (k >> 1) + 16 * g;
  const int chunks = (k + 127) >> 7;  // of 128 k
  uint4 cw[kDepth][NT];
  auto load = [&](int d, int c) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
      cw[d][t] = c * 128 + 32 * g < k ? *reinterpret_cast<const uint4*>(codes[t] + 64 * static_cast<long>(c)) : uint4{0, 0, 0, 0};
  };
  if (tid == 0) bad = 0;

  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{};

  const int per_stage = (kc >> 7) / job.wk;  // chunks per wave
  for (int k0 = 0, i0 = 0; k0 < k; k0 += kc, i0 += per_stage) {
    __syncthreads();  // the last stage's reads are done (and `bad` is cleared)
#pragma unroll
    for (int d = 0; d < kDepth; ++d)  // (underway while the inputs are laid out)
      if (d < per_stage) load(d, wave_k + (i0 + d) * job.wk);
    const int g0 = k0 / a.group;
    // inputs: 8 elements at a time
    const int eights = kc >> 3;
    for (int i = tid; i < nb * eights; i += 256) {
      const int r = i / eights, e = (i - r * eights) * 8;
      const long at = static_cast<long>(b0 + r) * k + k0 + e;
      const bool in = k0 + e < k;
      if (a.parts == 1) {
        uint4 v = in ? *reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.x) + at) : uint4{0, 0, 0, 0};
        // not finite: an exponent of ones in either half
        auto odd = [](unsigned u) { return (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u; };
        if (odd(v.x) || odd(v.y) || odd(v.z) || odd(v.w)) atomicOr(&bad, 1u << (r & 31));
        uint4 o;
        o.x = __builtin_amdgcn_perm(v.z, v.x, 0x05040100u);
        o.y = __builtin_amdgcn_perm(v.z, v.x, 0x07060302u);
        o.z = __builtin_amdgcn_perm(v.w, v.y, 0x05040100u);
        o.w = __builtin_amdgcn_perm(v.w, v.y, 0x07060302u);
        *reinterpret_cast<uint4*>(lds + r * xs + 2 * e) = o;
      } else {
        float v[8];
        if (!in) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        } else if (a.x_dtype == IRIS_F32) {
          load8(static_cast<const float*>(a.x) + at, v);
        } else {
          load8(static_cast<const bf16*>(a.x) + at, v);
        }
        bool odd = false;
        if (a.in_act == IRIS_ACT_SILU && in) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = silu(v[j]);
        }
        unsigned part[3][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          odd |= (bits_of(v[j]) & 0x7f800000u) == 0x7f800000u;
          part[0][j] = bits_of(v[j]) >> 16;
          const float r1 = v[j] - of_bits(part[0][j] << 16);
          part[1][j] = bits_of(r1) >> 16;
          part[2][j] = bits_of(r1 - of_bits(part[1][j] << 16)) >> 16;
        }
        if (odd) atomicOr(&bad, 1u << (r & 31));
#pragma unroll
        for (int s = 0; s < 3; ++s)
          *reinterpret_cast<uint4*>(lds + (s * nb + r) * xs + 2 * e) =
              uint4{part[s][0] | part[s][4] << 16, part[s][1] | part[s][5] << 16, part[s][2] | part[s][6] << 16,
                    part[s][3] | part[s][7] << 16};
      }
    }
    // scales and offsets of this stage's groups
    const int gn = min((min(k0 + kc, k) - 1) / a.group - g0 + 1, gs);
    for (int i = tid; i < n_wg * gn; i += 256) {
      const int r = i / gn, q = i - r * gn;
      const long at = static_cast<long>(min(n0 + r, n - 1)) * a.groups + g0 + q;
      const float scale = load_any(job.scales, a.scales_dtype, at);
      const float off = job.zeros ? -16.0f - static_cast<float>(job.zeros[at]) : -24.0f;
      const unsigned h = bits_of(off) >> 16;  // (exact: an integer below 2^8)
      sc[r * gs + q] = uint2{bits_of(scale), h | h << 16};
    }
    __syncthreads();

    auto chunk = [&](int d, int c, bool more) {
      // [row][128 k] of each lane group's 32 k to [k-step of 32][lane group's 8 k]
      unsigned u[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const auto p = __builtin_amdgcn_permlane32_swap(cw[d][t].x, cw[d][t].z, false, false);
        const auto q = __builtin_amdgcn_permlane32_swap(cw[d][t].y, cw[d][t].w, false, false);
        const auto r = __builtin_amdgcn_permlane16_swap(p[0], q[0], false, false);
        const auto s = __builtin_amdgcn_permlane16_swap(p[1], q[1], false, false);
        u[t][0] = r[0], u[t][1] = r[1], u[t][2] = s[0], u[t][3] = s[1];
      }
      if (more) load(d, c + kDepth * job.wk);
      const int kl = c * 128 - k0;  // in the stage
#pragma unroll
      for (int s0 = 0; s0 < 4; s0 += SPG) {
        const int q = (c * 128 + 32 * s0) / a.group - g0;
        f32x4 part[MT][NT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t) part[m][t] = f32x4{};
        uint2 sz[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) sz[t] = sc[((wave_n * NT + t) * 16 + l16) * gs + min(q, gn - 1)];
#pragma unroll
        for (int s = s0; s < s0 + SPG; ++s) {
          bf16x8 af[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m)
            af[m] = *reinterpret_cast<const bf16x8*>(lds + min(m * 16 + l16, rows - 1) * xs + 2 * (kl + 32 * s + 8 * g));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const unsigned v = u[t][s];
            const uint4 b4{(v << 3 & 0x00780078u) | 0x41804180u, (v >> 1 & 0x00780078u) | 0x41804180u,
                           (v >> 5 & 0x00780078u) | 0x41804180u, (v >> 9 & 0x00780078u) | 0x41804180u};
            const uint4 o4{sz[t].y, sz[t].y, sz[t].y, sz[t].y};
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              part[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[m], __builtin_bit_cast(bf16x8, b4), part[m][t], 0, 0, 0);
              part[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[m], __builtin_bit_cast(bf16x8, o4), part[m][t], 0, 0, 0);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][t][e] = __builtin_fmaf(of_bits(sz[t].x), part[m][t][e], acc[m][t][e]);
      }
    };
    for (int i = 0; i < per_stage; i += kDepth) {
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int c = wave_k + (i0 + i + d) * job.wk;
        if (i + d < per_stage && c < chunks) chunk(d, c, i + d + kDepth < per_stage);
      }
    }
  }

  // sums to LDS: [wave_k][weight row][A row + 1]
  __syncthreads();
  float* const red = reinterpret_cast<float*>(lds);
  const int rs = MT * 16 + 1;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(wave_k * n_wg + (wave_n * NT + t) * 16 + l16) * rs + m * 16 + 4 * g + e] = acc[m][t][e];
  __syncthreads();
  // y[b][row], in place of the first wave's sums (each read and written by one thread)
  for (int i = tid; i < nb * n_wg; i += 256) {
    const int b = i / n_wg, r = i - b * n_wg;
    float y = 0.0f;
    for (int s = a.parts - 1; s >= 0; --s)
      for (int q = 0; q < job.wk; ++q) y += red[(q * n_wg + r) * rs + s * nb + b];
    red[r * rs + b] = y;
  }
  __syncthreads();
  if (bad) {  // a row holding NaN or an infinity: its products one by one, as the formula has them
    for (int i = w; i < nb * n_wg; i += 4) {
      const int b = i / n_wg, r = i - b * n_wg;
      if (!(bad >> (b & 31) & 1) || n0 + r >= n) continue;
      const long row = n0 + r;
      float y = 0.0f;
      for (int e = lane; e < k; e += kWave) {
        const long q = row * a.groups + e / a.group;
        const unsigned code = job.codes[row * (k >> 1) + (e >> 1)] >> (4 * (e & 1)) & 15u;
        const float wv = load_any(job.scales, a.scales_dtype, q) *
                         (static_cast<float>(code) - (job.zeros ? static_cast<float>(job.zeros[q]) : 8.0f));
        float xv = load_any(a.x, a.x_dtype, static_cast<long>(b0 + b) * k + e);
        if (a.in_act == IRIS_ACT_SILU) xv = silu(xv);
        y = __builtin_fmaf(wv, xv, y);
      }
      y = wave_sum(y);
      if (lane == 0) red[r * rs + b] = y;
    }
    __syncthreads();
  }
  const int copies = job.n_extra ? job.n_extra : 1;
  for (int i = tid; i < nb * n_wg; i += 256) {
    const int b = i / n_wg, r = i - b * n_wg;
    const int row = n0 + r;
    if (row >= n) continue;
    float y = red[r * rs + b];
    if (job.bias) y += job.bias[row];
    if (a.out_act == IRIS_ACT_SILU) y = silu(y);
    for (int j = 0; j < copies; ++j) {
      const float v = job.n_extra ? y + job.extra[static_cast<long>(j) * n + row] : y;
      const long at = (static_cast<long>(j) * a.batch + b0 + b) * n + row;
      if (a.out_dtype == IRIS_F32)
        static_cast<float*>(job.out)[at] = v;
      else
        static_cast<bf16*>(job.out)[at] = from_f32<bf16>(v);
    }
  }
}

template <int MT, int NT, int SPG>
int launch_tiles(W4Launch& a, int jobs, hipStream_t stream) {
  // four weight tiles per workgroup where that gives every CU a workgroup, else one with k dealt to the waves
  // (by the product's own rows, so that a result does not depend on the other product of a launch)
  size_t lds = 0;
  int blocks[2] = {0, 0};
  for (int j = 0; j < jobs; ++j) {
    W4Job& job = a.job[j];
    job.wk = job.n >= 64L * NT * device_cus() ? 1 : 4;
    const int n_wg = 4 / job.wk * NT * 16;
    const int step = 128 * job.wk;
    auto bytes = [&](int kc) { return a.nb * a.parts * x_stride(kc) + n_wg * stage_groups(kc, a.group) * 8; };
    job.kc = (a.k + step - 1) / step * step;
    if (bytes(job.kc) > kLdsBytes) {
      job.kc = step;
      while (bytes(job.kc + step) <= kLdsBytes) job.kc += step;
    }
    const size_t need[2] = {static_cast<size_t>(bytes(job.kc)), static_cast<size_t>(job.wk) * n_wg * (MT * 16 + 1) * 4};
    lds = need[0] > lds ? need[0] : lds;
    lds = need[1] > lds ? need[1] : lds;
    blocks[j] = (job.n + n_wg - 1) / n_wg;
  }
  a.blocks0 = blocks[0];
  const dim3 grid(blocks[0] + blocks[1], (a.batch + a.nb - 1) / a.nb);
  IRIS_REQUIRE(grid.y < 65536, "gemv_w4: batch too large");
  gemv_w4_kernel<MT, NT, SPG><<<grid, 256, lds, stream>>>(a);
  return check_launch("gemv_w4");
}

template <int SPG>
int launch_rows(W4Launch& a, int jobs, hipStream_t stream) {
  // input rows in equal parts of at most kMaxRows A rows
  const int most = a.parts == 1 ? 32 : kMaxRows / a.parts;
  const int pieces = (a.batch + most - 1) / most;
  a.nb = (a.batch + pieces - 1) / pieces;
  switch ((a.nb * a.parts + 15) / 16) {
    case 1: return launch_tiles<1, 1, SPG>(a, jobs, stream);
    case 2: return launch_tiles<2, 1, SPG>(a, jobs, stream);
    default: return launch_tiles<3, 1, SPG>(a, jobs, stream);
  }
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_gemv_w4(const iris_gemv_w4_args* args, hipStream_t stream) {
  IRIS_REQUIRE(args, "gemv_w4: null pointer");
  const iris_gemv_w4_args& g = *args;
  IRIS_REQUIRE(g.jobs == 1 || g.jobs == 2, "gemv_w4: takes one or two products");
  IRIS_REQUIRE(g.batch >= 0 && g.batch < (1L << 20) && (g.x || g.batch == 0), "gemv_w4: bad batch or input");
  IRIS_REQUIRE(g.group > 0 && g.group % 32 == 0 && g.group < (1L << 30), "gemv_w4: the group must be a multiple of 32 (got %ld)",
               g.group);
  IRIS_REQUIRE((g.x_dtype == IRIS_F32 || g.x_dtype == IRIS_BF16) && (g.out_dtype == IRIS_F32 || g.out_dtype == IRIS_BF16) &&
                   (g.scales_dtype == IRIS_F32 || g.scales_dtype == IRIS_BF16),
               "gemv_w4: unknown dtype");
  IRIS_REQUIRE((g.in_act == IRIS_ACT_NONE || g.in_act == IRIS_ACT_SILU) &&
                   (g.out_act == IRIS_ACT_NONE || g.out_act == IRIS_ACT_SILU),
               "gemv_w4: unknown activation");
  IRIS_REQUIRE(g.k > 0 && g.k % 32 == 0 && g.k <= (1 << 20), "gemv_w4: need k %% 32 == 0 and k <= 2^20");
  IRIS_REQUIRE(aligned(g.x, 16), "gemv_w4: x must be 16-byte aligned");
  W4Launch a{};
  for (int j = 0; j < g.jobs; ++j) {
    const iris_gemv_w4_job& t = g.job[j];
    IRIS_REQUIRE(t.n > 0 && t.n < (1L << 30), "gemv_w4: bad weight rows");
    IRIS_REQUIRE(t.n_extra >= 0 && t.n_extra < (1L << 20) && (t.n_extra == 0 || t.extra_bias),
                 "gemv_w4: extra biases missing");
    IRIS_REQUIRE(t.codes && t.scales && (t.out || g.batch == 0), "gemv_w4: null pointer");
    IRIS_REQUIRE(aligned(t.codes, 16), "gemv_w4: codes must be 16-byte aligned");
    const char* out = static_cast<const char*>(t.out);
    const char* x = static_cast<const char*>(g.x);
    const long out_bytes = (t.n_extra ? t.n_extra : 1) * g.batch * t.n * (g.out_dtype == IRIS_F32 ? 4 : 2);
    const long x_bytes = g.batch * g.k * (g.x_dtype == IRIS_F32 ? 4 : 2);
    IRIS_REQUIRE(out + out_bytes <= x || x + x_bytes <= out, "gemv_w4: out must lie apart from x");
    a.job[j] = W4Job{static_cast<const unsigned char*>(t.codes),
                     t.scales,
                     static_cast<const unsigned char*>(t.zeros),
                     static_cast<int>(t.n),
                     t.bias,
                     t.extra_bias,
                     static_cast<int>(t.n_extra),
                     t.out};
  }
  if (g.batch == 0) return IRIS_OK;
  a.x = g.x;
  a.x_dtype = static_cast<int>(g.x_dtype);
  a.out_dtype = static_cast<int>(g.out_dtype);
  a.scales_dtype = static_cast<int>(g.scales_dtype);
  a.batch = static_cast<int>(g.batch);
  a.k = static_cast<int>(g.k);
  a.group = static_cast<int>(g.group);
  a.groups = static_cast<int>((g.k + g.group - 1) / g.group);
  a.in_act = static_cast<int>(g.in_act);
  a.out_act = static_cast<int>(g.out_act);
  a.parts = a.x_dtype == IRIS_BF16 && a.in_act == IRIS_ACT_NONE ? 1 : 3;
  const int jobs = static_cast<int>(g.jobs);
  if (a.group % 128 == 0) return launch_rows<4>(a, jobs, stream);
  if (a.group % 64 == 0) return launch_rows<2>(a, jobs, stream);
  return launch_rows<1>(a, jobs, stream);
}
