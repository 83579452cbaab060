// Matrix-vector products with 4-bit weights and group scales, for the calls of a few rows that gemv.hip
// serves with BF16 weights.
//
// W[n, k] = scale[n, k / group] (code[n, k] - zero[n, k / group]), codes 0..15 (element k of a row is the
// low half of byte k / 2 where k is even, the high half where it is odd), zero 8 where none are given;
// y[b, n] = act_out(sum_k W[n, k] act_in(x[b, k]) + bias[n]), out[j, b, n] = y[b, n] + extra_bias[j, n].
#include "iris_common.hpp"

namespace iris {
namespace {

constexpr int kMaxBatch = 4;

struct W4Job {
  const unsigned char* codes;
  const void* scales;
  const unsigned char* zeros;
  int n;
  const float *bias, *extra;
  int n_extra;
  void* out;
};
struct W4Launch {
  W4Job job;
  const void* x;
  int x_dtype, out_dtype, scales_dtype;
  int b0, nb, batch, k, group, groups, in_act, out_act;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, long i) {
  return dtype == IRIS_F32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const bf16*>(p)[i]);
}

// One wave per weight row; lane l has the bytes l, l + 64, ..
__global__ __launch_bounds__(256) void gemv_w4_kernel(W4Launch a) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.job.n) return;
  const int lane = threadIdx.x & 63;
  const unsigned char* codes = a.job.codes + static_cast<long>(row) * (a.k / 2);
  float acc[kMaxBatch] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = lane; i < a.k / 2; i += kWave) {
    const long g = static_cast<long>(row) * a.groups + 2 * i / a.group;
    const float scale = load_any(a.job.scales, a.scales_dtype, g);
    const float zero = a.job.zeros ? static_cast<float>(a.job.zeros[g]) : 8.0f;
    const float w0 = scale * (static_cast<float>(codes[i] & 15) - zero);
    const float w1 = scale * (static_cast<float>(codes[i] >> 4) - zero);
    for (int b = 0; b < a.nb; ++b) {
      const long at = static_cast<long>(a.b0 + b) * a.k + 2 * i;
      float x0 = load_any(a.x, a.x_dtype, at), x1 = load_any(a.x, a.x_dtype, at + 1);
      if (a.in_act == IRIS_ACT_SILU) x0 = silu(x0), x1 = silu(x1);
      acc[b] += w0 * x0 + w1 * x1;
    }
  }
  for (int b = 0; b < a.nb; ++b) {
    float y = wave_sum(acc[b]);
    if (lane != 0) continue;
    if (a.job.bias) y += a.job.bias[row];
    if (a.out_act == IRIS_ACT_SILU) y = silu(y);
    const int copies = a.job.n_extra ? a.job.n_extra : 1;
    for (int j = 0; j < copies; ++j) {
      const float v = a.job.n_extra ? y + a.job.extra[static_cast<long>(j) * a.job.n + row] : y;
      const long at = (static_cast<long>(j) * a.batch + a.b0 + b) * a.job.n + row;
      if (a.out_dtype == IRIS_F32)
        static_cast<float*>(a.job.out)[at] = v;
      else
        static_cast<bf16*>(a.job.out)[at] = from_f32<bf16>(v);
    }
  }
}

int check_job(const W4Job& job, int batch, int k) {
  IRIS_REQUIRE(job.n > 0 && k > 0 && k % 32 == 0 && k <= (1 << 20), "gemv_w4: need k %% 32 == 0 and k <= 2^20");
  IRIS_REQUIRE(job.n_extra >= 0 && (job.n_extra == 0 || job.extra), "gemv_w4: extra biases missing");
  IRIS_REQUIRE(job.codes && job.scales && (job.out || batch == 0), "gemv_w4: null pointer");
  IRIS_REQUIRE(aligned(job.codes, 16), "gemv_w4: codes must be 16-byte aligned");
  return IRIS_OK;
}

}  // namespace
}  // namespace iris

using namespace iris;

extern "C" int iris_gemv_w4(int jobs, const void* const* codes, const void* const* scales, int scales_dtype,
                            const void* const* zeros, int group, const void* x, int x_dtype, int batch, const int* n,
                            int k, const float* const* bias, const float* const* extra_bias, const int* n_extra,
                            void* const* out, int out_dtype, int in_act, int out_act, hipStream_t stream) {
  IRIS_REQUIRE((jobs == 1 || jobs == 2) && codes && scales && zeros && n && bias && extra_bias && n_extra && out,
               "gemv_w4: takes one or two products");
  IRIS_REQUIRE(batch >= 0 && (x || batch == 0), "gemv_w4: bad batch or input");
  IRIS_REQUIRE(group > 0 && group % 32 == 0, "gemv_w4: the group must be a multiple of 32 (got %d)", group);
  IRIS_REQUIRE((x_dtype == IRIS_F32 || x_dtype == IRIS_BF16) && (out_dtype == IRIS_F32 || out_dtype == IRIS_BF16) &&
                   (scales_dtype == IRIS_F32 || scales_dtype == IRIS_BF16),
               "gemv_w4: unknown dtype");
  IRIS_REQUIRE((in_act == IRIS_ACT_NONE || in_act == IRIS_ACT_SILU) &&
                   (out_act == IRIS_ACT_NONE || out_act == IRIS_ACT_SILU),
               "gemv_w4: unknown activation");
  W4Launch a{};
  a.x = x;
  a.x_dtype = x_dtype;
  a.out_dtype = out_dtype;
  a.scales_dtype = scales_dtype;
  a.batch = batch;
  a.k = k;
  a.group = group;
  a.groups = (k + group - 1) / group;
  a.in_act = in_act;
  a.out_act = out_act;
  W4Job job[2];
  for (int j = 0; j < jobs; ++j) {
    job[j] = W4Job{static_cast<const unsigned char*>(codes[j]),
                   scales[j],
                   static_cast<const unsigned char*>(zeros[j]),
                   n[j],
                   bias[j],
                   extra_bias[j],
                   n_extra[j],
                   out[j]};
    const int rc = check_job(job[j], batch, k);
    if (rc) return rc;
  }
  for (int j = 0; j < jobs; ++j)
    for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
      a.job = job[j];
      a.b0 = b0;
      a.nb = batch - b0 < kMaxBatch ? batch - b0 : kMaxBatch;
      gemv_w4_kernel<<<dim3((a.job.n + 3) / 4), 256, 0, stream>>>(a);
      const int rc = check_launch("gemv_w4");
      if (rc) return rc;
    }
  return IRIS_OK;
}
