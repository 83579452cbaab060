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
//   offset leaves by a second MFMA of the same A with -(16 + zero) in every place, exact like the first.
//   What the FP32 sums hold is thus x (16 + code) and -x (16 + zero), up to 62 |x| scale a weight whatever
//   code - zero is, and their roundings are to that: an input far above the others leaves about 2^-24 of it
//   times 24 scale in results that its weight, a zero, has no part in (inputs of 1000 to 10000 among ones of 1,
//   meeting zeros alone in 1312 x 150 weights: up to 2e-4 of the result in norm; without such inputs 0.9e-7).
// - A: BF16 rows as they are; FP32 rows (and activated ones) as three BF16 rows that add up to them exactly
//   (8 + 8 + 8 bits of significand, by truncation; below 2^-110 the last row's steps of 2^-133 cut them off), so
//   FP32 inputs keep FP32 products at no extra MFMA while
//   three rows per input row fit 16. They lie in LDS with each 8 elements in the order 0 4 1 5 2 6 3 7 that
//   the codes come in.
// - The FP32 sums of a group of at least 32 are scaled and added to the row's FP32 sums.
// A workgroup's eight waves are dealt over weight tiles and over k (their sums joined in LDS): many tiles where
// the weight has rows enough for all CUs, because every workgroup lays out all inputs anew, few where it has not.
// One row, 131072 x 4096: 60 us, 4.6 TB/s (a large copy moves 4.9). Small calls are bound by their chain of latencies:
// inputs and scales to LDS, products, the join of the waves, the store: 6.2 us for 2560 x 2560 of which a launch that
// does nothing takes about 3; 12.0 us for two FP32 rows, 15360 x 2560, 24 outputs (VALU issue 26 % of the waves' cycles,
// the matrix cores busy 10 %); 15.1 us for 24 rows, 13696 x 2560 (26 and 15 %). More rows than a workgroup holds read and
// unpack all codes once per piece: 13696 x 2560, BF16 32 rows 17 us, 33: 23, 64: 32; FP32 16 rows 20, 17: 24, 64: 73.
#include "iris_common.hpp"

namespace iris {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kMaxRows = 48;  // A rows of a workgroup
constexpr int kAhead = 8;     // extra biases of a thread that are loaded at the start
constexpr int kScaleItems = 8;  // scales of a thread and stage
// LDS of a workgroup (inputs and scales of all k, or of two stages of k) where a CU holds two of them, and at most
constexpr size_t kLdsTwo = 78 << 10, kLdsOne = 156 << 10;

struct W4Job {
  const unsigned char* codes;
  const void* scales;
  const unsigned char* zeros;
  int n;
  const float *bias, *extra;
  int n_extra;
  void* out;
  int wn;  // waves side by side over weight rows; the other kWaves / wn - 1 share their k
  int kc;  // k per stage, a multiple of 128 kWaves / wn
};
struct W4Launch {
  W4Job job[2];
  int blocks0;
  const void* x;
  int out_dtype, scales_f32;
  int batch, nb;  // input rows in all, and per workgroup (blockIdx.y)
  int k, group, groups, in_act, out_act;
  unsigned group_steps, group_magic;  // group / 32 and 2^32 / that + 1
};

__device__ __forceinline__ unsigned bits_of(float x) { return __builtin_bit_cast(unsigned, x); }
__device__ __forceinline__ float of_bits(unsigned x) { return __builtin_bit_cast(float, x); }

// The group of 32-wide k-step s.
__device__ __forceinline__ int group_of(const W4Launch& a, int s) {
  return a.group_steps == 1 ? s : static_cast<int>(__umulhi(static_cast<unsigned>(s), a.group_magic));
}

// i / d and the remainder of 0 <= i < 2^22 by d's reciprocal.
struct Divisor {
  int d;
  float inv;
  __device__ __forceinline__ explicit Divisor(int by) : d(by), inv(__builtin_amdgcn_rcpf(static_cast<float>(by))) {}
  __device__ __forceinline__ void operator()(int i, int& q, int& r) const {
    q = static_cast<int>(static_cast<float>(i) * inv);
    r = i - q * d;
    if (r < 0) --q, r += d;
    if (r >= d) ++q, r -= d;
  }
};

// LDS of a launch: A rows of kc BF16 + 16 bytes (the 16 rows of a fragment read then start in distinct banks),
// and per weight row and group of a stage the scale and the offset's BF16 pair, rows an odd number of pairs apart.
__host__ __device__ __forceinline__ int x_stride(int kc) { return 2 * kc + 16; }
__host__ __device__ __forceinline__ int stage_groups(int kc, int group) { return ((kc + group - 1) / group + 1) | 1; }

// 8-element inputs of a thread and stage, by the 16-byte words that they take.
template <typename X>
constexpr int input_items() { return sizeof(X) == 2 ? 8 : 4; }

// X: the inputs' type; PARTS: A rows per input row, 1, or 3 for FP32 and activated inputs; MT tiles of 16 A rows, NT
// of 16 weight rows per wave; SPG 32-wide k-steps per scale; DEPTH code loads (NT of 16 rows x 128 k each) underway
// per wave, which divides a stage's chunks of a wave where there are several stages (STAGED). Without stages nothing
// of a next one waits in registers, and two workgroups share a CU (one row, 65536 x 4096: 39 us staged, 32 whole).
template <typename X, int PARTS, int MT, int NT, int SPG, int DEPTH, bool STAGED>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(MT == 1 && !STAGED ? 4 : 2))) void
gemv_w4_kernel(W4Launch a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int odd;
  constexpr int XI = input_items<X>();
  const bool second = static_cast<int>(blockIdx.x) >= a.blocks0;
  W4Job job = a.job[0];
  if (second) job = a.job[1];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = job.wn, wk = kWaves / wn, wave_n = w & (wn - 1), wave_k = w / wn;
  const int n_wg = wn * NT * 16;  // a power of two
  const int n0 = (static_cast<int>(blockIdx.x) - (second ? a.blocks0 : 0)) * n_wg;
  const int b0 = blockIdx.y * a.nb;
  const int nb = min(a.nb, a.batch - b0);
  const int rows = nb * PARTS;
  const int k = a.k, kc = job.kc, n = job.n;
  const int xs = x_stride(kc), gs = stage_groups(kc, a.group);
  const int stage_bytes = a.nb * PARTS * xs + n_wg * gs * 8;  // A rows, then [n_wg][gs] scales and offsets

  // codes, in chunks of 128 k dealt to the waves; past the row's end the last ones again: their inputs are zeros
  const unsigned char* codes[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
    codes[t] = job.codes + static_cast<long>(min(n0 + (wave_n * NT + t) * 16 + l16, n - 1)) * (k >> 1) + 16 * g;
  const int chunks = (k + 127) >> 7;
  uint4 cw[DEPTH][NT];
  auto load = [&](int d, int c) {
    const int at = min(c * 64, (k >> 1) - 16 - 16 * g);
#pragma unroll
    for (int t = 0; t < NT; ++t) cw[d][t] = *reinterpret_cast<const uint4*>(codes[t] + at);
  };

  // A stage's scales and inputs: loaded into registers (while the stage before is computed), then laid out.
  const int most_r = n - 1 - n0;
  const char* const scale_at = static_cast<const char*>(job.scales) + static_cast<long>(n0) * a.groups * (a.scales_f32 ? 4 : 2);
  const unsigned char* const zero_at = job.zeros + static_cast<long>(n0) * a.groups;
  unsigned scale[kScaleItems], zero[kScaleItems];
  auto stage_group = [&](int k0, int& g0, int& gn) {  // the first of a stage's groups and their number
    g0 = group_of(a, k0 >> 5);
    gn = min(group_of(a, (min(k0 + kc, k) - 1) >> 5) - g0 + 1, gs);
  };
  auto load_scales = [&](int k0, int from) {
    int g0, gn;
    stage_group(k0, g0, gn);
    const Divisor by_gn(gn);
    int at[kScaleItems];
#pragma unroll
    for (int u = 0; u < kScaleItems; ++u) {
      int r, q;
      by_gn(min(from + tid + u * kThreads, n_wg * gn - 1), r, q);
      at[u] = min(r, most_r) * a.groups + g0 + q;
    }
    if (a.scales_f32) {
#pragma unroll
      for (int u = 0; u < kScaleItems; ++u)
        if (from + w * 64 + u * kThreads < n_wg * gn) scale[u] = *reinterpret_cast<const unsigned*>(scale_at + 4L * at[u]);
    } else {
#pragma unroll
      for (int u = 0; u < kScaleItems; ++u)
        if (from + w * 64 + u * kThreads < n_wg * gn) scale[u] = *reinterpret_cast<const unsigned short*>(scale_at + 2L * at[u]);
    }
    if (job.zeros) {
#pragma unroll
      for (int u = 0; u < kScaleItems; ++u)
        if (from + w * 64 + u * kThreads < n_wg * gn) zero[u] = zero_at[at[u]];
    }
  };
  auto lay_scales = [&](int k0, char* stage, int from) {
    uint2* const sc = reinterpret_cast<uint2*>(stage + a.nb * PARTS * xs);
    int g0, gn;
    stage_group(k0, g0, gn);
    const Divisor by_gn(gn);
#pragma unroll
    for (int u = 0; u < kScaleItems; ++u)
      if (from + w * 64 + u * kThreads < n_wg * gn) {  // (whole waves; past the last item, it again)
        int r, q;
        by_gn(min(from + tid + u * kThreads, n_wg * gn - 1), r, q);
        // (exact: an integer below 2^8)
        const unsigned h = bits_of(-16.0f - (job.zeros ? static_cast<float>(zero[u]) : 8.0f)) >> 16;
        sc[r * gs + q] = uint2{a.scales_f32 ? scale[u] : scale[u] << 16, h | h << 16};
      }
  };
  const int eights = kc >> 3, items = nb * eights;
  const Divisor by_eights(eights);
  const X* const x_at = static_cast<const X*>(a.x) + static_cast<long>(b0) * k;
  constexpr int XW = sizeof(X) / 2;  // 16-byte words of an item
  uint4 xr[XI][XW];
  auto load_inputs = [&](int k0, int from) {
#pragma unroll
    for (int u = 0; u < XI; ++u)
      if (from + w * 64 + u * kThreads < items) {
        int r, e;
        by_eights(min(from + tid + u * kThreads, items - 1), r, e);
        const uint4* x = reinterpret_cast<const uint4*>(x_at + r * k + min(k0 + 8 * e, k - 8));
#pragma unroll
        for (int i = 0; i < XW; ++i) xr[u][i] = x[i];
      }
  };
  auto lay_inputs = [&](int k0, char* stage, int from) {
#pragma unroll
    for (int u = 0; u < XI; ++u)
      if (from + w * 64 + u * kThreads < items) {
        int r, e;
        by_eights(min(from + tid + u * kThreads, items - 1), r, e);
        e *= 8;
        const unsigned keep = k0 + e < k ? ~0u : 0u;
        uint4 v = xr[u][0];
        v = uint4{v.x & keep, v.y & keep, v.z & keep, v.w & keep};
        if constexpr (PARTS == 1) {
          uint4 o;
          o.x = __builtin_amdgcn_perm(v.z, v.x, 0x05040100u);
          o.y = __builtin_amdgcn_perm(v.z, v.x, 0x07060302u);
          o.z = __builtin_amdgcn_perm(v.w, v.y, 0x05040100u);
          o.w = __builtin_amdgcn_perm(v.w, v.y, 0x07060302u);
          *reinterpret_cast<uint4*>(stage + r * xs + 2 * e) = o;
        } else {
          float x[8];
          if constexpr (sizeof(X) == 4) {
            const uint4 z = xr[u][XW - 1];
            x[0] = of_bits(v.x), x[1] = of_bits(v.y), x[2] = of_bits(v.z), x[3] = of_bits(v.w);
            x[4] = of_bits(z.x & keep), x[5] = of_bits(z.y & keep), x[6] = of_bits(z.z & keep), x[7] = of_bits(z.w & keep);
          } else {
            x[0] = of_bits(v.x << 16), x[1] = of_bits(v.x & 0xffff0000u), x[2] = of_bits(v.y << 16), x[3] = of_bits(v.y & 0xffff0000u);
            x[4] = of_bits(v.z << 16), x[5] = of_bits(v.z & 0xffff0000u), x[6] = of_bits(v.w << 16), x[7] = of_bits(v.w & 0xffff0000u);
          }
          if (a.in_act == IRIS_ACT_SILU) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = silu(x[j]);  // (0 past k stays 0)
          }
          unsigned part[3][8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            part[0][j] = bits_of(x[j]) >> 16;
            const float r1 = x[j] - of_bits(part[0][j] << 16);
            part[1][j] = bits_of(r1) >> 16;
            part[2][j] = bits_of(r1 - of_bits(part[1][j] << 16)) >> 16;
          }
#pragma unroll
          for (int s = 0; s < 3; ++s)
            *reinterpret_cast<uint4*>(stage + (s * nb + r) * xs + 2 * e) =
                uint4{part[s][0] | part[s][4] << 16, part[s][1] | part[s][5] << 16, part[s][2] | part[s][6] << 16,
                      part[s][3] | part[s][7] << 16};
        }
      }
  };

  load_scales(0, 0);
  load_inputs(0, 0);
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(d, wave_k + d * wk);
  // the output's row of this thread (n_wg divides the threads) and its first biases, underway from the start too
  const int out_r = tid & (n_wg - 1), out_row = n0 + out_r, out_at = min(out_row, n - 1);
  const int step = kThreads / n_wg, first = tid / n_wg;
  const int outs = (job.n_extra ? job.n_extra : 1) * nb;  // (copy j, input row b), j major
  const Divisor by_nb(nb);
  const float bias = job.bias ? job.bias[out_at] : 0.0f;
  float ahead[kAhead] = {};
  if (job.n_extra) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      int j, b;
      by_nb(min(first + u * step, outs - 1), j, b);
      ahead[u] = job.extra[static_cast<long>(j) * n + out_at];
    }
  }
  lay_scales(0, lds, 0);
  lay_inputs(0, lds, 0);
  if constexpr (!STAGED) {  // (what the first registers did not hold)
    for (int from = kScaleItems * kThreads; from < n_wg * gs; from += kScaleItems * kThreads) {
      load_scales(0, from);
      lay_scales(0, lds, from);
    }
    for (int from = XI * kThreads; from < items; from += XI * kThreads) {
      load_inputs(0, from);
      lay_inputs(0, lds, from);
    }
  }
  lds_barrier();

  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[m][t] = f32x4{};
  // (kept in registers, one of each kind: as literals they would split every and-or in two)
  unsigned mask = 0x00780078u, sixteen = 0x41804180u;
  asm volatile("" : "+s"(mask), "+v"(sixteen));
  int a_row[MT];  // LDS offset of this lane's A rows (those past the last repeat it)
#pragma unroll
  for (int m = 0; m < MT; ++m) a_row[m] = min(m * 16 + l16, rows - 1) * xs;
  const int per_stage = (kc >> 7) / wk;  // chunks per wave
  const int mine = (chunks - wave_k + wk - 1) / wk;  // of this wave in all
  char* stage = lds;
  for (int k0 = 0, i0 = 0; k0 < k; k0 += kc, i0 += per_stage) {
    const bool more = STAGED && k0 + kc < k;
    if (more) {
      load_scales(k0 + kc, 0);
      load_inputs(k0 + kc, 0);
    }
    const uint2* const sc = reinterpret_cast<const uint2*>(stage + a.nb * PARTS * xs);
    int g0, gn;
    stage_group(k0, g0, gn);
    auto chunk = [&](int d, int c, bool next) {
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
      if (next) load(d, c + DEPTH * wk);
      const int kl = c * 128 - k0;  // in the stage
      constexpr int SG = 4 / SPG;   // scales of the chunk
      uint2 sz[SG][NT];
#pragma unroll
      for (int q = 0; q < SG; ++q) {
        const int at = min(group_of(a, c * 4 + SPG * q) - g0, gn - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) sz[q][t] = sc[((wave_n * NT + t) * 16 + l16) * gs + at];
      }
      f32x4 part[SG][MT][NT];
#pragma unroll
      for (int q = 0; q < SG; ++q)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t) part[q][m][t] = f32x4{};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int q = s / SPG;
        bf16x8 af[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
          af[m] = *reinterpret_cast<const bf16x8*>(stage + a_row[m] + 2 * (kl + 32 * s + 8 * g));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const unsigned v = u[t][s], z = sz[q][t].y;
          const uint4 b4{(v << 3 & mask) | sixteen, (v >> 1 & mask) | sixteen, (v >> 5 & mask) | sixteen,
                         (v >> 9 & mask) | sixteen};
          const uint4 o4{z, z, z, z};
#pragma unroll
          for (int m = 0; m < MT; ++m)
            part[q][m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[m], __builtin_bit_cast(bf16x8, o4), part[q][m][t], 0, 0, 0);
#pragma unroll
          for (int m = 0; m < MT; ++m)
            part[q][m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[m], __builtin_bit_cast(bf16x8, b4), part[q][m][t], 0, 0, 0);
        }
      }
#pragma unroll
      for (int q = 0; q < SG; ++q)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[m][t][e] = __builtin_fmaf(of_bits(sz[q][t].x), part[q][m][t][e], acc[m][t][e]);
      __builtin_amdgcn_sched_barrier(0);  // (one chunk's registers at a time)
    };
    // this wave's chunks of the stage; the ring's loads stand in straight code (a branch around one would wait for
    // it) and run on into the next stage's
    const int here = min(mine - i0, per_stage);
    int i = 0;
    for (; i + DEPTH <= here; i += DEPTH)
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) chunk(d, wave_k + (i0 + i + d) * wk, true);
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
      if (i + d < here) chunk(d, wave_k + (i0 + i + d) * wk, false);
    if (more) {
      stage = stage == lds ? lds + stage_bytes : lds;  // (its last readers are a barrier behind)
      lay_scales(k0 + kc, stage, 0);
      lay_inputs(k0 + kc, stage, 0);
      lds_barrier();
    }
  }

  // sums to LDS: [wave_k][weight row][A row + 1]
  lds_barrier();
  if (tid == 0) odd = 0;
  float* const red = reinterpret_cast<float*>(lds);
  const int rs = MT * 16 + 1;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(wave_k * n_wg + (wave_n * NT + t) * 16 + l16) * rs + m * 16 + 4 * g + e] = acc[m][t][e];
  lds_barrier();
  // y[row][b], in place of the first wave's sums (each read and written by one thread)
  bool finite = true;
  for (int b = first; b < nb; b += step) {
    float y = 0.0f;
    for (int s = PARTS - 1; s >= 0; --s) {
      float v[kWaves];
#pragma unroll
      for (int q = 0; q < kWaves; ++q) v[q] = red[(min(q, wk - 1) * n_wg + out_r) * rs + s * nb + b];
#pragma unroll
      for (int q = 0; q < kWaves; ++q) y += q < wk ? v[q] : 0.0f;
    }
    finite = finite && __builtin_isfinite(y);
    red[out_r * rs + b] = y;
  }
  if (!finite) odd = 1;
  lds_barrier();
  // NaN or an infinity among the inputs (or scales): the offset's products turn it into NaN, so such sums are taken
  // product by product, as the formula has them
  if (odd) {
    for (int i = w; i < nb * n_wg; i += kWaves) {
      const int b = i / n_wg, r = i - b * n_wg;
      if (n0 + r >= n || __builtin_isfinite(red[r * rs + b])) continue;
      const long row = n0 + r;
      float y = 0.0f;
      for (int e = lane; e < k; e += kWave) {
        const long q = row * a.groups + e / a.group;
        const unsigned code = job.codes[row * (k >> 1) + (e >> 1)] >> (4 * (e & 1)) & 15u;
        const float wv = (a.scales_f32 ? static_cast<const float*>(job.scales)[q] : to_f32(static_cast<const bf16*>(job.scales)[q])) *
                         (static_cast<float>(code) - (job.zeros ? static_cast<float>(job.zeros[q]) : 8.0f));
        float xv = to_f32(static_cast<const X*>(a.x)[static_cast<long>(b0 + b) * k + e]);
        if (a.in_act == IRIS_ACT_SILU) xv = silu(xv);
        y = __builtin_fmaf(wv, xv, y);
      }
      y = wave_sum(y);
      if (lane == 0) red[r * rs + b] = y;
    }
    lds_barrier();
  }
  if (out_row >= n) return;
  auto store = [&](long at, float v) {
    if (a.out_dtype == IRIS_F32)
      static_cast<float*>(job.out)[at] = v;
    else
      static_cast<bf16*>(job.out)[at] = from_f32<bf16>(v);
  };
  auto finish = [&](int i, float add) {
    int j, b;
    by_nb(i, j, b);
    float y = red[out_r * rs + b];
    if (job.bias) y += bias;
    if (a.out_act == IRIS_ACT_SILU) y = silu(y);
    if (job.n_extra) y += add;
    store((static_cast<long>(j) * a.batch + b0 + b) * n + out_row, y);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (first + u * step < outs) finish(first + u * step, ahead[u]);
  for (int i = first + kAhead * step; i < outs; i += step)
    finish(i, job.n_extra ? job.extra[static_cast<long>(i / nb) * n + out_row] : 0.0f);
}

// One product's share of a launch: waves over weight rows and k per stage for `depth` code loads underway; 0 where
// that depth does not fit.
template <typename X, int PARTS, int MT, int NT>
size_t plan_job(const W4Launch& a, W4Job& job, int& blocks, int depth) {
  auto bytes = [&](int wn, int kc) {  // of a stage
    return static_cast<size_t>(a.nb) * PARTS * x_stride(kc) + static_cast<size_t>(wn) * NT * 16 * stage_groups(kc, a.group) * 8;
  };
  auto whole = [&](int wn) { return (a.k + 128 * (kWaves / wn) - 1) / (128 * (kWaves / wn)) * (128 * (kWaves / wn)); };
  // as many weight rows per workgroup as leave four of five CUs a workgroup (by the product's own rows, so that a
  // result does not depend on the other product of a launch; twice the workgroups of half the rows, us: 2 FP32 rows,
  // 15360 x 2560 12.5 instead of 11.9, 15360 x 5120 26.8 / 15.7; 24 BF16 rows, 13696 x 2560 24.6 / 14.8), and half of
  // that where a CU then holds two (one row, 32768 x 8192: 33.8 instead of 39.9; where all of k only then is one stage
  // it loses: 4 FP32 rows, 32768 x 4096 27.8 / 23.8)
  constexpr int kLeast = MT > 2 ? 2 : 1;
  job.wn = kWaves;
  while (job.wn > kLeast && 5L * job.n < 4L * job.wn * NT * 16 * device_cus()) job.wn /= 2;
  if (job.wn > kLeast && bytes(job.wn, whole(job.wn)) > kLdsTwo && bytes(job.wn / 2, whole(job.wn / 2)) <= kLdsTwo) job.wn /= 2;
  const int n_wg = job.wn * NT * 16, wk = kWaves / job.wn;
  blocks = (job.n + n_wg - 1) / n_wg;
  const size_t sums = static_cast<size_t>(wk) * n_wg * (MT * 16 + 1) * 4;
  size_t lds = bytes(job.wn, whole(job.wn));
  if (lds <= kLdsOne) {
    job.kc = whole(job.wn);
  } else {
    auto fits = [&](int kc) {  // (a stage's inputs and scales are in registers while the stage before is computed)
      return a.nb * (kc / 8) <= input_items<X>() * kThreads && n_wg * stage_groups(kc, a.group) <= kScaleItems * kThreads &&
             2 * bytes(job.wn, kc) <= kLdsOne;
    };
    const int unit = 128 * wk * depth;
    if (!fits(unit)) return 0;
    for (job.kc = unit; fits(job.kc + unit);) job.kc += unit;
    lds = 2 * bytes(job.wn, job.kc);
  }
  return lds > sums ? lds : sums;
}

// Launches with DEPTH code loads underway, if that fits; 1 where it does not. (staged: every product in stages of k.)
template <typename X, int PARTS, int MT, int NT, int SPG, int DEPTH>
int launch_depth(W4Launch& a, int jobs, bool staged, hipStream_t stream) {
  size_t lds = 0;
  int blocks[2] = {0, 0};
  for (int j = 0; j < jobs; ++j) {
    const size_t need = plan_job<X, PARTS, MT, NT>(a, a.job[j], blocks[j], DEPTH);
    if (need == 0 || (!staged && a.job[j].kc < a.k)) return 1;
    lds = need > lds ? need : lds;
  }
  a.blocks0 = blocks[0];
  const dim3 grid(blocks[0] + blocks[1], (a.batch + a.nb - 1) / a.nb);
  IRIS_REQUIRE(grid.y < 65536 && grid.x < (1u << 23), "gemv_w4: too many input or weight rows");
  if (staged)
    gemv_w4_kernel<X, PARTS, MT, NT, SPG, DEPTH, true><<<grid, kThreads, lds, stream>>>(a);
  else if constexpr (DEPTH > 1)
    gemv_w4_kernel<X, PARTS, MT, NT, SPG, DEPTH, false><<<grid, kThreads, lds, stream>>>(a);
  return check_launch("gemv_w4");
}

template <typename X, int PARTS, int MT, int NT, int SPG>
int launch_tiles(W4Launch& a, int jobs, hipStream_t stream) {
  // A kernel in stages lays out what one round of its registers holds, one for all of k more than that: a product of
  // each kind take a launch each.
  if (jobs == 2) {
    bool whole[2];
    for (int j = 0; j < 2; ++j) {
      int blocks;
      whole[j] = plan_job<X, PARTS, MT, NT>(a, a.job[j], blocks, 1) && a.job[j].kc >= a.k;
    }
    if (whole[0] != whole[1]) {
      W4Launch second = a;
      second.job[0] = a.job[1];
      const int rc = launch_tiles<X, PARTS, MT, NT, SPG>(a, 1, stream);
      return rc ? rc : launch_tiles<X, PARTS, MT, NT, SPG>(second, 1, stream);
    }
  }
  // (more registers spill; with two workgroups on a CU two loads a wave do as well as four: 15360 x 5120 15.7 / 16.3 us)
  constexpr int kDepth = MT == 1 ? 4 : 2;
  int rc = launch_depth<X, PARTS, MT, NT, SPG, 2>(a, jobs, false, stream);
  if (rc == 1) rc = launch_depth<X, PARTS, MT, NT, SPG, kDepth>(a, jobs, true, stream);
  if (rc == 1) rc = launch_depth<X, PARTS, MT, NT, SPG, 1>(a, jobs, true, stream);
  return rc == 1 ? fail(IRIS_E_UNSUPPORTED, "gemv_w4: no stage of k fits") : rc;  // (one of 128 k per wave always does)
}

template <typename X, int PARTS, int SPG>
int launch_rows(W4Launch& a, int jobs, hipStream_t stream) {
  // input rows in equal parts of at most kMaxRows A rows
  const int most = PARTS == 1 ? 32 : kMaxRows / PARTS;
  const int pieces = (a.batch + most - 1) / most;
  a.nb = (a.batch + pieces - 1) / pieces;
  switch ((a.nb * PARTS + 15) / 16) {
    case 1: return launch_tiles<X, PARTS, 1, 1, SPG>(a, jobs, stream);
    case 2: return launch_tiles<X, PARTS, 2, 2, SPG>(a, jobs, stream);
    default:
      if constexpr (PARTS == 3) return launch_tiles<X, PARTS, 3, 2, SPG>(a, jobs, stream);
      return IRIS_E_INVALID;  // (32 rows at most)
  }
}

template <typename X, int PARTS>
int launch_groups(W4Launch& a, int jobs, hipStream_t stream) {
  return a.group % 64 == 0 ? launch_rows<X, PARTS, 2>(a, jobs, stream) : launch_rows<X, PARTS, 1>(a, jobs, stream);
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
    IRIS_REQUIRE(t.n_extra >= 0 && t.n_extra < (1L << 16) && (t.n_extra == 0 || t.extra_bias),
                 "gemv_w4: extra biases missing, or 65536 and more");
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
  if (g.jobs == 2) {
    const char* first = static_cast<const char*>(g.job[0].out);
    const char* second = static_cast<const char*>(g.job[1].out);
    auto bytes = [&](int j) { return (g.job[j].n_extra ? g.job[j].n_extra : 1) * g.batch * g.job[j].n * (g.out_dtype == IRIS_F32 ? 4 : 2); };
    IRIS_REQUIRE(first + bytes(0) <= second || second + bytes(1) <= first, "gemv_w4: the products' outputs must lie apart");
  }
  a.x = g.x;
  a.out_dtype = static_cast<int>(g.out_dtype);
  a.batch = static_cast<int>(g.batch);
  a.k = static_cast<int>(g.k);
  a.group = static_cast<int>(g.group);
  a.groups = static_cast<int>((g.k + g.group - 1) / g.group);
  // (k / 32 <= 2^15 and group / 32 cut to that: the product's error stays below 2^32)
  a.group_steps = static_cast<unsigned>(g.group < (1 << 20) ? g.group / 32 : 1 << 15);
  a.group_magic = static_cast<unsigned>((1ull << 32) / a.group_steps) + 1;
  a.in_act = static_cast<int>(g.in_act);
  a.out_act = static_cast<int>(g.out_act);
  const int jobs = static_cast<int>(g.jobs);
  a.scales_f32 = g.scales_dtype == IRIS_F32;
  if (g.x_dtype == IRIS_F32) return launch_groups<float, 3>(a, jobs, stream);
  return a.in_act == IRIS_ACT_NONE ? launch_groups<bf16, 1>(a, jobs, stream) : launch_groups<bf16, 3>(a, jobs, stream);
}
