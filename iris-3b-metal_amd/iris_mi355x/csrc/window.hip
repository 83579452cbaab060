// Attention with a sliding window and a few first tokens that stay visible, 128-wide heads with grouped
// K/V heads: whole prompts, and one or a few queries over a long cache.
//
// Query t of batch item b stands at position p = start[b] + t. Key j < length[b] is visible to it iff
//   (no causal limit or j <= p) and (no window or |p - j| < window or j < sinks) and key_mask[b, j] != 0,
// so a query's keys are [0, sink_end) and [low, high) less the masked ones (Span). The result is
//   o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m) over its visible keys (m their largest
//   score), and 0 where nothing is visible.
//
// One pass over the keys with a running maximum and sum, tile by tile (Attend): S^T = K Q^T and O^T = V^T P^T
// on v_mfma_f32_16x16x32_bf16, a lane owning one query and four keys of every 16, so that P^T stays in the
// registers it was computed in. K and V arrive as rows (views of a projection or a cache) and go straight
// into LDS; V^T fragments are read from the V rows by the transposing LDS read (four rows by 16 columns per
// 16 lanes). Only tiles that hold a visible key of some query of the workgroup are visited.
//
// window_attn_kernel (prompts): bound by the MFMAs and the softmax beside them. A workgroup's waves share a
// ring of K/V tiles; a wave is one query head's 16 or 32 rows, the heads of a K/V head side by side. 8192 tokens, 32 on 8
// heads, window 4096: 398 us, 1037 TFLOP/s of visible pairs, the matrix cores busy 51 % of the cycles in which a CU holds
// waves and a wave issuing VALU 27 % of its own; 4352 tokens, 20 on 5, two-sided window 640 and 256 first keys: 87 us, 713
// TFLOP/s (680 workgroups in 512 places: CUs hold waves for 68 % of the launch); small prompts are a chain of 5 us and
// 0.8 us per tile. (Replayed in a graph; a profiler's single launches take 434 and 97 us.)
// window_few_kernel (few queries): bound by the keys' and values' way from memory. The rows of a tile are the
// (query, head) pairs of one K/V head; every wave streams key tiles of its own through its own LDS, without
// barriers, and the waves' and workgroups' parts are joined at the end (window_join_kernel for the latter). 16 queries
// of 32 on 8 heads over 65536 keys at most: 598 us, 5.5 TB/s; one query over 1028 keys: 11 us in two launches. Several row
// tiles of a K/V head each read its keys: 16 queries of 20 on 5 heads over a cache of 32768 keys 45 us, 32: 98, where K
// and V read once are 17.
// window_rows_kernel: row strides of 2^24 elements and more, too large for the 32-bit offsets of the others.
#include "iris_common.hpp"

#include <type_traits>

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
  int hpw, rows_per_wg, n_qblocks, n_hgroups;  // window_attn_kernel
  int total_wg;
  int splits, row_tiles;  // window_few_kernel
  float *part_o, *part_ml;  // [row][split][128] and [row][split][2] of the split form
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

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

// Lane i of 16 gets column i of the 4 x 16 block whose row j the lanes 4 j .. 4 j + 3 address, 8 bytes each.
__device__ __forceinline__ bf16x4 read_tr(const char* p) {
  return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

// The bytes of `rows` rows of 128 values `stride` elements apart as a buffer: reads past them give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const bf16* p, long rows, long stride) {
  const long bytes = rows <= 0 ? 0 : (rows - 1) * stride * 2 + 2 * kHd;
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, static_cast<int>(bytes < 0x7fffffffL ? bytes : 0x7fffffffL),
                                           kBufferFlags);
}

// 16-byte chunk c of row r of a tile lies at chunk c ^ swz of that row in LDS: the 16 rows of a K fragment read
// (one chunk each) and the 8 rows that 32 lanes of a transposing V read touch (two chunks each) then start in
// distinct banks.
__device__ __forceinline__ int k_swz(int row) { return row & 15; }
__device__ __forceinline__ int v_swz(int row) { return 2 * (row & 7); }

// The running attention of 16 RB queries of one head per wave over tiles of KVT keys in LDS (K rows, V rows, 256 bytes
// each). Lane l (l16 = l % 16, h = l / 16) owns queries 16 qb + l16 and, of each 16 keys, keys 4 h .. 4 h + 3:
// s[kb][qb][e] is key 16 kb + 4 h + e. A P V step of 32 keys takes them in the order 16 (j / 4) + 4 h + j % 4 for
// k-index 8 h + j, in P^T and V^T alike. o[db][qb][e] is dim 16 db + 4 h + e.
template <int RB, int KVT>
struct Attend {
  static constexpr int NKB = KVT / 16, H32 = KVT / 32;
  bf16x8 qf[RB][4];  // query 16 qb + l16, dims 32 st + 8 h .. + 8
  f32x4 o[8][RB];
  float m[RB], l[RB];  // log2 domain; l: this lane's keys only
  Span span[RB];
  int k_rd[4], v_rd[8];  // LDS offsets of the fragment reads by k-step and dim block
  int l16, h;
  float sl2;  // > 0

  // The scale's sign goes into the queries (and a scale of 0 turns them into zeros).
  __device__ __forceinline__ void load_query(int qb, const bf16* row, float scale_log2) {
    sl2 = scale_log2 == 0.0f ? 1.0f : __builtin_fabsf(scale_log2);
    const unsigned flip = scale_log2 < 0.0f ? 0x80008000u : 0u, keep = scale_log2 == 0.0f ? 0u : ~0u;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      uint4 v = *reinterpret_cast<const uint4*>(row + 32 * st + 8 * h);
      v = uint4{(v.x ^ flip) & keep, (v.y ^ flip) & keep, (v.z ^ flip) & keep, (v.w ^ flip) & keep};
      qf[qb][st] = __builtin_bit_cast(bf16x8, v);
    }
  }
  __device__ __forceinline__ void start(int lane) {
    l16 = lane & 15, h = lane >> 4;
#pragma unroll
    for (int st = 0; st < 4; ++st) k_rd[st] = l16 * 256 + 16 * ((4 * st + h) ^ k_swz(l16));
    const int row = 4 * h + (l16 >> 2);
#pragma unroll
    for (int db = 0; db < 8; ++db)
      v_rd[db] = row * 256 + 16 * ((2 * db + ((l16 & 3) >> 1)) ^ v_swz(row)) + 8 * (l16 & 1);
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int qb = 0; qb < RB; ++qb) m[qb] = -INFINITY, l[qb] = 0.0f;
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < RB; ++qb) o[db][qb] = f32x4{};
  }
  // Whether some output is not finite.
  __device__ __forceinline__ bool odd() const {
    float x = 0.0f;
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int qb = 0; qb < RB; ++qb)
#pragma unroll
        for (int e = 0; e < 4; ++e) x = __builtin_fmaf(o[db][qb][e], 0.0f, x);
    return x != 0.0f;  // (NaN)
  }
  __device__ __forceinline__ bool visible(int qb, int j, unsigned long long keys, int in_tile) const {
    return (j < span[qb].sink_end || (j >= span[qb].low && j < span[qb].high)) && (keys >> in_tile & 1);
  }
  __device__ __forceinline__ bf16x8 v_frag(const char* vl, int hf, int db) const {
    const char* p = vl + hf * 32 * 256 + v_rd[db];
    const bf16x4 a = read_tr(p), b = read_tr(p + 16 * 256);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  // partial: some query may not see some key; `keys` has a bit for every key of the tile that the key mask shows.
  // careful: values that are not finite may be among the tile's.
  // K: the tile's K rows in LDS, or its K fragments (i = NKB st + kb) in registers.
  template <typename K>
  __device__ __forceinline__ void tile(K kl, const char* vl, int kv0, bool partial, unsigned long long keys, bool careful) {
    // S^T, K fragments from LDS read four ahead of their MFMAs; at a raised priority, so that a wave in its MFMAs is
    // picked before those of its SIMD that are in their softmax
    constexpr int NK = 4 * NKB;
    constexpr bool kLds = std::is_same<K, const char*>::value;
    f32x4 s[NKB][RB];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int qb = 0; qb < RB; ++qb) s[kb][qb] = f32x4{};
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kLds) {
      bf16x8 kf[4];
      auto read_k = [&](int i) { kf[i % 4] = *reinterpret_cast<const bf16x8*>(kl + (i % NKB) * 16 * 256 + k_rd[i / NKB]); };
#pragma unroll
      for (int i = 0; i < 4; ++i) read_k(i);
#pragma unroll
      for (int i = 0; i < NK; ++i) {
#pragma unroll
        for (int qb = 0; qb < RB; ++qb)
          s[i % NKB][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i % 4], qf[qb][i / NKB], s[i % NKB][qb], 0, 0, 0);
        if (i + 4 < NK) read_k(i + 4);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads
#pragma unroll
      for (int i = 0; i + 4 < NK; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, RB, 0);  // MFMAs
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4 * RB, 0);
    } else {
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int qb = 0; qb < RB; ++qb)
          s[i % NKB][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kl[i], qf[qb][i / NKB], s[i % NKB][qb], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);

    if (partial) {
      // (selects, not branches: the bounds of a query relative to this lane's first key)
      const unsigned long long mine = keys >> (4 * h);
      const unsigned bits[2] = {static_cast<unsigned>(mine), static_cast<unsigned>(mine >> 32)};
      const int j0 = kv0 + 4 * h;
#pragma unroll
      for (int qb = 0; qb < RB; ++qb) {
        const int from = j0 - span[qb].low, sinks = span[qb].sink_end - j0;
        const unsigned width = max(span[qb].high - span[qb].low, 0);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 16 * kb + e;
            const int seen = (static_cast<int>(i < sinks) | static_cast<int>(static_cast<unsigned>(from + i) < width)) &
                             static_cast<int>(bits[i / 32] >> (i % 32) & 1u);
            s[kb][qb][e] = seen ? s[kb][qb][e] : -INFINITY;
          }
      }
    }

    // Online softmax against a running maximum that is raised lazily: while a lane's exponentials of the tile add
    // up to at most 2^8 the maximum and the output stay as they are; otherwise the queries that need it take their
    // exact maxima, rescale, and recompute. A query with no key so far keeps -inf, and its hidden keys are taken
    // against 0, which makes them exact zeros instead of NaN. The sums add the FP32 exponentials; P is rounded to
    // BF16 (the MFMA's operand; a second one for the rest would double the P V products) after that: up to 2^-8 of
    // each weight, and 0.0020 to 0.0023 from a 64-bit result in norm where FP32 weights leave 0.0016, the output's rounding.
    bf16x8 pf[H32][RB];
    auto probs = [&](int qb, float ref) {
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][qb][e], sl2, -ref));
          pf[kb / 2][qb][4 * (kb % 2) + e] = from_f32<bf16>(x);
          sum += x;
        }
      return sum;
    };
#pragma unroll
    for (int qb = 0; qb < RB; ++qb) {
      float sum = probs(qb, m[qb]);
      const int need = !(sum <= 256.0f);  // also for NaN (the first tile, a hidden key of a query without keys)
      if (__any(need)) {
        int raise = need | __shfl_xor(need, 16);
        raise |= __shfl_xor(raise, 32);
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[kb][qb][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = raise ? fmaxf(m[qb], mx * sl2) : m[qb];
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m[qb] - ref);  // exactly 1 unless raised
        l[qb] *= alpha;
#pragma unroll
        for (int db = 0; db < 8; ++db) o[db][qb] *= alpha;
        m[qb] = m_new;
        sum = probs(qb, ref);
      }
      l[qb] += sum;
    }
    if (careful) {
      // A value that is not finite reaches every query of the MFMA (0 times NaN): where some query does not see the
      // tile whole, it is left out of the products and added to the queries that see it.
#pragma unroll
      for (int i = 0; i < 8 * H32; ++i) {
        bf16x8 v = v_frag(vl, i / 8, i % 8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (partial && !__builtin_isfinite(to_f32(v[e]))) v[e] = from_f32<bf16>(0.0f);
#pragma unroll
        for (int qb = 0; qb < RB; ++qb)
          o[i % 8][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pf[i / 8][qb], o[i % 8][qb], 0, 0, 0);
      }
      if (!partial) return;
#pragma unroll 1
      for (int key = 0; key < KVT; ++key)
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          const int d = 16 * db + 4 * h;
          const f32x4 v = load4(reinterpret_cast<const bf16*>(vl + key * 256 + 16 * ((d >> 3) ^ v_swz(key)) + 2 * (d & 7)));
#pragma unroll
          for (int qb = 0; qb < RB; ++qb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!__builtin_isfinite(v[e]) && visible(qb, kv0 + key, keys, key)) o[db][qb][e] += v[e];
        }
      return;
    }
    // O^T, the V^T fragments (i = 8 hf + db) read four ahead of their MFMAs
    constexpr int NV = 8 * H32;
    bf16x8 vf[4];
    auto read_v = [&](int i) { vf[i % 4] = v_frag(vl, i / 8, i % 8); };
#pragma unroll
    for (int i = 0; i < 4; ++i) read_v(i);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int qb = 0; qb < RB; ++qb)
        o[i % 8][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[i % 4], pf[i / 8][qb], o[i % 8][qb], 0, 0, 0);
      if (i + 4 < NV) read_v(i + 4);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (int i = 0; i + 4 < NV; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, RB, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4 * RB, 0);
  }

  // A tile, if some query between those of the spans a and z sees a key of it.
  template <bool MASK, typename K>
  __device__ __forceinline__ void visit(const Span& a, const Span& z, K kl, const char* vl, int kv0,
                                        unsigned long long keys, bool careful) {
    constexpr unsigned long long kAll = KVT == 64 ? ~0ull : (1ull << (KVT & 63)) - 1;
    // (none of it: below the windows and past the first keys, or past the windows)
    if (kv0 >= z.sink_end && (kv0 >= z.high || kv0 + KVT <= a.low)) return;
    if (MASK && !(keys & kAll)) return;
    const bool all = kv0 + KVT <= a.sink_end || (kv0 >= z.low && kv0 + KVT <= a.high);
    tile(kl, vl, kv0, !all || (MASK && (keys & kAll) != kAll), keys, careful);
  }
};

// The tiles that hold a visible key of queries at positions first .. last: those of [0, sinks), then those of
// [low, high) that are not among them.
template <int KVT>
struct Tiles {
  int sink, band, count;
  __device__ __forceinline__ Tiles(const WindowArgs& p, long first, long last, int length) {
    const Span a = span_of(p, first, length), z = span_of(p, last, length);
    sink = (z.sink_end + KVT - 1) / KVT;
    band = max(a.low / KVT, sink);
    count = sink + max((z.high + KVT - 1) / KVT - band, 0);
    if (a.low >= z.high) count = sink;
  }
  __device__ __forceinline__ int key(int t) const { return (t < sink ? t : t - sink + band) * KVT; }
};
// A bit for every key of the tile at kv0 that the mask shows, from one byte per lane.
__device__ __forceinline__ int mask_byte(const unsigned char* mask, int kv0, int lane, int length) {
  return kv0 + lane < length ? mask[kv0 + lane] : 0;
}

// Waves of a workgroup, keys of a tile and tiles of the ring.
constexpr int kPromptWaves = 4, kPromptKeys = 64, kPromptStages = 2;

template <int RB, bool MASK>
__global__ __launch_bounds__(64 * kPromptWaves) __attribute__((amdgpu_waves_per_eu(2))) void
window_attn_kernel(WindowArgs p) {
  constexpr int NW = kPromptWaves, KVT = kPromptKeys, STAGES = kPromptStages;
  constexpr int STAGE = 2 * KVT * 256;  // bytes: K rows, then V rows
  constexpr int LOADS = KVT / 4 / NW;   // 1 KB loads (4 rows) per wave and operand
  constexpr int LPW = 2 * LOADS;
  static_assert(LOADS * 4 * NW == KVT && STAGES >= 2 && (STAGES - 2) * LPW < 64, "pipeline");
  // (the only LDS of the kernel: with a second object, a fence's included, the compiler waits for the prefetch before
  // every tile's reads)
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE];

  // logical workgroup: (item, K/V head, head group) major, query block minor and, where later queries see more
  // keys, the last block first; one K/V head's blocks stay on one XCD
  int wg = xcd_remap(blockIdx.x, p.total_wg);
  int qblk = wg % p.n_qblocks;
  if (p.causal) qblk = p.n_qblocks - 1 - qblk;
  wg /= p.n_qblocks;
  const int hg = wg % p.n_hgroups;
  wg /= p.n_hgroups;
  const int kvh = wg % p.kv_heads;
  const int b = wg / p.kv_heads;

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hd = kvh * (p.heads / p.kv_heads) + hg * p.hpw + w % p.hpw;
  const int length = __builtin_amdgcn_readfirstlane(item_length(p, b));
  const long pos0 = item_start(p, b, length);
  const int wg0 = qblk * p.rows_per_wg;
  const int q0 = wg0 + (w / p.hpw) * 16 * RB;

  Attend<RB, KVT> at;
  at.start(lane);
#pragma unroll
  for (int qb = 0; qb < RB; ++qb) {
    const int row = min(q0 + 16 * qb + at.l16, p.n_q - 1);
    at.load_query(qb, p.q + b * p.qs_b + hd * p.qs_h + row * p.qs_n, p.scale_log2);
    at.span[qb] = span_of(p, pos0 + row, length);
  }
  const Tiles<KVT> tiles(p, pos0 + wg0, pos0 + min(wg0 + p.rows_per_wg, p.n_q) - 1, length);
  const Span first = span_of(p, pos0 + min(q0, p.n_q - 1), length), last = span_of(p, pos0 + min(q0 + 16 * RB - 1, p.n_q - 1), length);
  const bool idle = q0 >= p.n_q;

  const bf16* kh = p.k + b * p.ks_b + kvh * p.ks_h;
  const bf16* vh = p.v + b * p.vs_b + kvh * p.vs_h;
  const unsigned char* mask = MASK ? p.key_mask + b * p.mask_stride : nullptr;
  int k_off[LOADS], v_off[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = (w * LOADS + j) * 4 + (lane >> 4);
    k_off[j] = r * static_cast<int>(p.ks_n) * 2 + 16 * ((lane & 15) ^ k_swz(r));
    v_off[j] = r * static_cast<int>(p.vs_n) * 2 + 16 * ((lane & 15) ^ v_swz(r));
  }
  const __amdgpu_buffer_rsrc_t rk = rows_buffer(kh, length, p.ks_n), rv = rows_buffer(vh, length, p.vs_n);
  auto issue = [&](int t, int stage) {
    const int kv0 = tiles.key(t);
    const int ks = kv0 * static_cast<int>(p.ks_n) * 2, vs = kv0 * static_cast<int>(p.vs_n) * 2;
    bf16* kl = reinterpret_cast<bf16*>(lds + stage * STAGE);
    bf16* vl = kl + KVT * kHd;
    if (kv0 + KVT <= length) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        buffer_load_lds16(rk, kl + (w * LOADS + j) * 512, k_off[j], ks);
        buffer_load_lds16(rv, vl + (w * LOADS + j) * 512, v_off[j], vs);
      }
    } else {  // the last key again in the rows past it
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int r = (w * LOADS + j) * 4 + (lane >> 4), back = max(r - (length - 1 - kv0), 0);
        buffer_load_lds16(rk, kl + (w * LOADS + j) * 512, k_off[j] - back * static_cast<int>(p.ks_n) * 2, ks);
        buffer_load_lds16(rv, vl + (w * LOADS + j) * 512, v_off[j] - back * static_cast<int>(p.vs_n) * 2, vs);
      }
    }
  };

  const int n_tiles = tiles.count;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    int byte = MASK && n_tiles > 0 ? mask_byte(mask, tiles.key(0), lane, length) : 0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < n_tiles) issue(s, s);
    for (int t = 0, stage = 0; t < n_tiles; ++t, stage = stage + 1 == STAGES ? 0 : stage + 1) {
      unsigned long long keys = ~0ull;
      if (MASK) {
        keys = __ballot(byte != 0);
        if (t + 1 < n_tiles) byte = mask_byte(mask, tiles.key(t + 1), lane, length);
      }
      if (t + STAGES - 2 < n_tiles)
        wait_vmcnt<(STAGES - 2) * LPW>();
      else
        wait_vmcnt<0>();
      __builtin_amdgcn_s_barrier();  // tile t is there; the stage of tile t - 1 is no longer read
      asm volatile("" ::: "memory");
      if (t + STAGES - 1 < n_tiles) issue(t + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
      const int kv0 = tiles.key(t);
      if (idle) continue;
      const char* kl = lds + stage * STAGE;
      at.template visit<MASK>(first, last, kl, kl + KVT * 256, kv0, keys, pass != 0);
    }
    // not finite: once more, keeping such values to the queries that see them
    if (pass == 1) break;
    int* const flags = reinterpret_cast<int*>(lds);
    lds_barrier();  // (the last tile is read)
    if (lane == 0) flags[w] = 0;
    if (at.odd()) flags[w] = 1;
    lds_barrier();
    int odd = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) odd |= flags[i];
    if (!odd) break;
    lds_barrier();
    at.clear();
  }

#pragma unroll
  for (int qb = 0; qb < RB; ++qb) {
    float l = at.l[qb] + __shfl_xor(at.l[qb], 16);
    l += __shfl_xor(l, 32);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int row = q0 + 16 * qb + at.l16;
    if (row >= p.n_q) continue;
    bf16* out = p.out + b * p.os_b + row * p.os_n + hd * kHd + 4 * at.h;
#pragma unroll
    for (int db = 0; db < 8; ++db) store4(out + 16 * db, at.o[db][qb] * inv);
  }
}

// Few queries: the 16 rows of a wave's tile are (query, head of the group) pairs r = t group + g of one K/V head. K
// fragments go straight to registers (a lane's row of 16 keys), V rows to the wave's ring in LDS.
constexpr int kFewWaves = 8, kFewKeys = 32;
constexpr int kMaxSplits = 64;

// Tiles of a split: whole rounds of the waves.
__host__ __device__ __forceinline__ int few_share(int tiles, int splits) {
  return (tiles + splits * kFewWaves - 1) / (splits * kFewWaves) * kFewWaves;
}

template <bool MASK>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2))) void window_few_kernel(WindowArgs p) {
  constexpr int KVT = kFewKeys, STAGE = KVT * 256, LOADS = KVT / 4;
  // (one object, as in window_attn_kernel: the V rings, two stages a wave; after the loop the waves' sums, then their
  // maxima)
  __shared__ __attribute__((aligned(1024))) char lds[kFewWaves * 2 * STAGE];
  float (*const ml)[16][2] = reinterpret_cast<float (*)[16][2]>(lds + kFewWaves * 16 * 132 * 4);

  int wg = xcd_remap(blockIdx.x, p.total_wg);
  const int rt = wg % p.row_tiles;
  wg /= p.row_tiles;
  const int split = wg % p.splits;
  wg /= p.splits;
  const int kvh = wg % p.kv_heads;
  const int b = wg / p.kv_heads;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = p.heads / p.kv_heads, rows = group * p.n_q;
  const int length = __builtin_amdgcn_readfirstlane(item_length(p, b));
  const long pos0 = item_start(p, b, length);
  const long pos_a = pos0 + rt * 16 / group, pos_z = pos0 + min(rt * 16 + 15, rows - 1) / group;
  const Span first = span_of(p, pos_a, length), last = span_of(p, pos_z, length);
  const Tiles<KVT> tiles(p, pos_a, pos_z, length);
  const int per = few_share(tiles.count, p.splits);
  const int t0 = split * per + w, end = min(tiles.count, (split + 1) * per);

  const bf16* kh = p.k + b * p.ks_b + kvh * p.ks_h;
  const bf16* vh = p.v + b * p.vs_b + kvh * p.vs_h;
  const unsigned char* mask = MASK ? p.key_mask + b * p.mask_stride : nullptr;
  Attend<1, KVT> at;
  at.start(lane);
  const int k_off = at.l16 * static_cast<int>(p.ks_n) * 2 + 16 * at.h;  // (a fragment: row l16 of 16 keys, 8 dims)
  int v_off[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = j * 4 + (lane >> 4);
    v_off[j] = r * static_cast<int>(p.vs_n) * 2 + 16 * ((lane & 15) ^ v_swz(r));
  }
  char* const mine = lds + w * 2 * STAGE;
  bf16x8 kf[2][8];
  int byte[2];
  // (STAGE-constant: the registers of the two stages; the K loads first, so that they are waited for alone)
  auto issue = [&](int t, int stage) {
    const int kv0 = tiles.key(t);
    const __amdgpu_buffer_rsrc_t rk = rows_buffer(kh + kv0 * p.ks_n, length - kv0, p.ks_n);
    const __amdgpu_buffer_rsrc_t rv = rows_buffer(vh + kv0 * p.vs_n, length - kv0, p.vs_n);
    const int half = 16 * static_cast<int>(p.ks_n) * 2;
    if (MASK) byte[stage] = mask_byte(mask, kv0, lane, length);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      kf[stage][i] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 64 * (i / 2) + (i % 2) * half, 0, 0));
    bf16* vl = reinterpret_cast<bf16*>(mine + stage * STAGE);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) buffer_load_lds16(rv, vl + j * 512, v_off[j], 0);
  };
  if (t0 < end) issue(t0, 0);
  const int row = min(rt * 16 + at.l16, rows - 1), t_row = row / group, hd = kvh * group + row - t_row * group;
  at.load_query(0, p.q + b * p.qs_b + hd * p.qs_h + t_row * p.qs_n, p.scale_log2);
  at.span[0] = span_of(p, pos0 + t_row, length);
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    if (pass == 1 && t0 < end) issue(t0, 0);
    for (int t = t0; t < end;) {
#pragma unroll
      for (int stage = 0; stage < 2; ++stage) {
        if (t >= end) break;
        if (t + kFewWaves < end) {
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the other stage's last reads are done
          issue(t + kFewWaves, stage ^ 1);
          wait_vmcnt<8 + LOADS>();
        } else {
          wait_vmcnt<0>();
        }
        asm volatile("" ::: "memory");
        const unsigned long long keys = MASK ? __ballot(byte[stage] != 0) : ~0ull;
        at.template visit<MASK>(first, last, &kf[stage][0], mine + stage * STAGE, tiles.key(t), keys, pass != 0);
        t += kFewWaves;
      }
    }
    if (pass == 1 || !__any(at.odd())) break;  // as in window_attn_kernel, each wave for itself
    at.clear();
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  }

  // join the waves: every wave's sums against the largest of their maxima, then one thread per 8 dims of a row
  float l = at.l[0] + __shfl_xor(at.l[0], 16);
  l += __shfl_xor(l, 32);
  lds_barrier();  // (the rings are no longer read)
  if (lane < 16) ml[w][lane][0] = at.m[0], ml[w][lane][1] = l;
  lds_barrier();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) top = fmaxf(top, ml[i][at.l16][0]);
  const float ref = top == -INFINITY ? 0.0f : top;
  const float mine_scale = __builtin_amdgcn_exp2f(at.m[0] - ref);
  float* const sums = reinterpret_cast<float*>(lds) + w * 16 * 132;  // rows of 132: distinct banks
#pragma unroll
  for (int db = 0; db < 8; ++db) store4(sums + at.l16 * 132 + 16 * db + 4 * at.h, at.o[db][0] * mine_scale);
  lds_barrier();
  const int r = threadIdx.x >> 4, d = (threadIdx.x & 15) * 8;
  if (r >= 16 || rt * 16 + r >= rows) return;
  float acc[8] = {}, lsum = 0.0f, rtop = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) rtop = fmaxf(rtop, ml[i][r][0]);
  const float rref = rtop == -INFINITY ? 0.0f : rtop;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) {
    float v[8];
    load8(reinterpret_cast<const float*>(lds) + (i * 16 + r) * 132 + d, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += v[e];
    lsum += ml[i][r][1] * __builtin_amdgcn_exp2f(ml[i][r][0] - rref);
  }
  const int rt_row = rt * 16 + r, tq = rt_row / group, hq = kvh * group + rt_row - tq * group;
  if (p.splits == 1) {
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
    bf16* out = p.out + b * p.os_b + tq * p.os_n + hq * kHd + d;
    store4(out, f32x4{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv});
    store4(out + 4, f32x4{acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv});
  } else {
    const long at_row = ((static_cast<long>(b) * p.heads + hq) * p.n_q + tq) * p.splits + split;
    store8(p.part_o + at_row * kHd + d, acc);
    if (d == 0) *reinterpret_cast<f32x2*>(p.part_ml + 2 * at_row) = f32x2{rtop, lsum};
  }
}

// One wave per (item, head, query): lane s has split s's maximum and sum, then dims 2 l and 2 l + 1.
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs p, long total) {
  const long row = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (row >= total) return;
  const int lane = threadIdx.x & 63;
  f32x2 ml = lane < p.splits ? *reinterpret_cast<const f32x2*>(p.part_ml + 2 * (row * p.splits + lane)) : f32x2{-INFINITY, 0.0f};
  float top = ml[0];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float ref = top == -INFINITY ? 0.0f : top;
  const float scale = __builtin_amdgcn_exp2f(ml[0] - ref);
  const float l = wave_sum(ml[1] * scale);
  const float* o = p.part_o + row * p.splits * kHd + 2 * lane;
  float o0 = 0.0f, o1 = 0.0f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const f32x2 v = *reinterpret_cast<const f32x2*>(o + s * kHd);
    const float f = __shfl(scale, s);
    o0 = __builtin_fmaf(v[0], f, o0);
    o1 = __builtin_fmaf(v[1], f, o1);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int t = static_cast<int>(row % p.n_q), h = static_cast<int>(row / p.n_q % p.heads), b = static_cast<int>(row / p.n_q / p.heads);
  bf16* out = p.out + b * p.os_b + t * p.os_n + h * kHd + 2 * lane;
  *reinterpret_cast<bf16x2*>(out) = bf16x2{from_f32<bf16>(o0 * inv), from_f32<bf16>(o1 * inv)};
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
    const float e = x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - top);  // (also while top is -inf)
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
  IRIS_REQUIRE(batch * heads * n_q < (1L << 31), "window_attn: need fewer than 2^31 rows of queries and heads");
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
  // (the stride of an axis of one says nothing)
  auto stride = [](const long* shape, const long* strides, int i) { return shape[i] > 1 ? strides[i] : (i == 2 ? kHd : 0); };
  p.qs_b = stride(g.q_shape, g.q_strides, 0), p.qs_h = stride(g.q_shape, g.q_strides, 1), p.qs_n = stride(g.q_shape, g.q_strides, 2);
  p.ks_b = stride(g.k_shape, g.k_strides, 0), p.ks_h = stride(g.k_shape, g.k_strides, 1), p.ks_n = stride(g.k_shape, g.k_strides, 2);
  p.vs_b = stride(g.v_shape, g.v_strides, 0), p.vs_h = stride(g.v_shape, g.v_strides, 1), p.vs_n = stride(g.v_shape, g.v_strides, 2);
  for (long x : {p.qs_b, p.qs_h, p.qs_n, p.ks_b, p.ks_h, p.ks_n, p.vs_b, p.vs_h, p.vs_n})
    IRIS_REQUIRE(x % 8 == 0 && x >= 0, "window_attn: strides must be multiples of 8 elements, and not negative");
  p.os_b = batch > 1 ? g.out_strides[0] : 0, p.os_n = n_q > 1 ? g.out_strides[1] : 0;
  IRIS_REQUIRE((n_q == 1 || p.os_n >= heads * kHd) && (batch == 1 || p.os_b >= heads * kHd) && p.os_b % 4 == 0 && p.os_n % 4 == 0,
               "window_attn: output rows must not overlap, strides must be multiples of 4");
  const StridedRuns out_rows = strided_runs(g.out, g.out_shape, g.out_strides, 2, 2, heads * kHd);
  IRIS_REQUIRE(!share_memory(out_rows, out_rows), "window_attn: output rows must not overlap");
  const void* in[3] = {g.q, g.k, g.v};
  const long* shapes[3] = {g.q_shape, g.k_shape, g.v_shape};
  const long* strides[3] = {g.q_strides, g.k_strides, g.v_strides};
  for (int i = 0; i < 3; ++i)
    IRIS_REQUIRE(!share_memory(out_rows, strided_runs(in[i], shapes[i], strides[i], 3, 2, kHd)),
                 "window_attn: out must lie apart from q, k and v");
  p.q = static_cast<const bf16*>(g.q);
  p.k = static_cast<const bf16*>(g.k);
  p.v = static_cast<const bf16*>(g.v);
  p.out = static_cast<bf16*>(g.out);
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.n_q = static_cast<int>(n_q);
  p.n_k = static_cast<int>(n_k);
  p.window = g.window < (1L << 60) ? g.window : (1L << 60);
  p.sinks = g.sinks < (1L << 60) ? g.sinks : (1L << 60);
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
// Which kernel a call takes, by its shapes alone.
enum { kRows, kPrompt, kFew };
int window_plan(WindowArgs& p) {
  const int group = p.heads / p.kv_heads, rows = group * p.n_q;
  if (p.ks_n >= (1L << 24) || p.vs_n >= (1L << 24)) return kRows;  // (32 rows of a tile by 32-bit offsets)
  p.hpw = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
  p.n_hgroups = group / p.hpw;
  p.row_tiles = (rows + 15) / 16;
  const long base = static_cast<long>(p.batch) * p.kv_heads * p.row_tiles, cus = device_cus();
  // Few: no more 16-row tiles than CUs, so that the prompts' form, a wave for 16 rows of a head with all of its keys,
  // would leave most waves of the card without work. us, few / prompts (heads of packed rows): 20 on 5 heads, 16 queries of
  // 32768 keys 68 / 605, 32: 101 / 575, 64 of 4096 keys: 26 / 61, 128 of 1000 (160 tiles): 16 / 18, of 16384: 135 / 224;
  // 8 on 1 head, 400 of 1000 (200): 15.5 / 18; beyond: 32 items of 16 queries, 1024 keys (640) 49 / 27; 64 items of one query, 2048 keys (320)
  // 81 / 68. (The prompts' form reaches all rows by 32-bit offsets; this one those of a tile.)
  if (base > cus && (p.n_k + 64) * (p.ks_n > p.vs_n ? p.ks_n : p.vs_n) * 2 < (1L << 31)) return kPrompt;
  // keys that a tile's queries can see at most, in tiles
  long keys = p.n_k;
  if (p.window) {
    const long queries = p.n_q < 15 / group + 2 ? p.n_q : 15 / group + 2;
    const long reach = (p.causal ? p.window : 2 * p.window - 1) + queries - 1 + 2 * kFewKeys, sinks = p.sinks + kFewKeys;
    keys = reach + sinks < keys ? reach + sinks : keys;
  }
  // as many workgroups as CUs, of one tile a wave (two rather than a second launch; one more than CUs is a second
  // round: 128 queries of 1000 keys 23 instead of 16 us); where every wave keeps 16 tiles, up to four for every CU.
  // us by the number of splits: one token, 20 on 5 heads, 1028 keys 1: 15.2, 4: 11.4, 8: 11.5, 16: 13.1; 4096 keys
  // 4: 20.4, 8: 16.0, 16: 15.6, 32: 17.7; 16384 keys 8: 32.6, 16: 24.6, 32: 22.9; 32 on 8 heads, 65536 keys 16: 82,
  // 32: 66, 64: 76; 16 items of 4096 keys 1: 76, 2: 59, 4: 59, 8: 65; of 65536 keys 1: 1077, 2: 781, 4: 749, 8: 727
  const long tiles = (keys + kFewKeys - 1) / kFewKeys;
  auto least = [](long a, long b) { return a < b ? a : b; };
  const long one = tiles <= 2 * kFewWaves ? 1 : least(cus / base, (tiles + kFewWaves - 1) / kFewWaves);
  const long four = least(4 * cus / base, tiles / (16 * kFewWaves));
  const long splits = one > four ? one : four;
  p.splits = static_cast<int>(splits < 1 ? 1 : splits > kMaxSplits ? kMaxSplits : splits);
  const int per = few_share(static_cast<int>(tiles), p.splits);
  if (per > 0) p.splits = static_cast<int>((tiles + per - 1) / per);
  return kFew;
}
long window_workspace(const WindowArgs& p) {
  return p.splits > 1 ? static_cast<long>(p.batch) * p.heads * p.n_q * p.splits * (kHd + 2) * 4 : 0;
}
}  // namespace

extern "C" int iris_window_attn_workspace(const iris_window_attn_args* args, long* bytes) {
  IRIS_REQUIRE(bytes, "window_attn: null pointer");
  *bytes = 0;
  WindowArgs p{};
  const int rc = window_args(args, p);
  if (rc || p.batch == 0) return rc;
  if (window_plan(p) == kFew) *bytes = window_workspace(p);
  return IRIS_OK;
}

extern "C" int iris_window_attn(const iris_window_attn_args* args, hipStream_t stream) {
  WindowArgs p{};
  const int rc = window_args(args, p);
  if (rc || p.batch == 0) return rc;
  const long rows = static_cast<long>(p.batch) * p.heads * p.n_q;
  const int plan = window_plan(p);
  IRIS_REQUIRE(plan == kPrompt || rows < (1L << 26), "window_attn: too many rows of queries and heads");
  if (plan == kRows) {
    window_rows_kernel<<<dim3(static_cast<unsigned>((rows + 3) / 4)), 256, 0, stream>>>(p, rows);
  } else if (plan == kPrompt) {
    // 32 rows a wave (a K/V fragment read from LDS serves two MFMAs) where that leaves seven workgroups for four CUs,
    // else 16 (twice the workgroups). 20 query heads on 5 K/V heads, us, 32 / 16 rows: causal 300 tokens 13.1 / 9.4,
    // 1000: 26.8 / 21.8, two of 1000: 34.9 / 29.5, eight of 300 (400 workgroups of 32 rows): 19.3 / 19.1, 4352 (680):
    // 138 / 150; all of 4352 to all 211 / 226; 32 on 8 heads, four of 512 (512): 24.5 / 24.8
    auto groups = [&](int rb) {
      p.rows_per_wg = 16 * rb * kPromptWaves / p.hpw;
      p.n_qblocks = (p.n_q + p.rows_per_wg - 1) / p.rows_per_wg;
      return static_cast<long>(p.batch) * p.kv_heads * p.n_hgroups * p.n_qblocks;
    };
    long total = groups(2);
    const bool few = 4 * total <= 7L * device_cus();
    if (few) total = groups(1);
    IRIS_REQUIRE(total < (1L << 24), "window_attn: too many rows of queries and heads");
    p.total_wg = static_cast<int>(total);
    const dim3 grid(p.total_wg);
    if (few) {
      if (p.key_mask)
        window_attn_kernel<1, true><<<grid, 64 * kPromptWaves, 0, stream>>>(p);
      else
        window_attn_kernel<1, false><<<grid, 64 * kPromptWaves, 0, stream>>>(p);
    } else {
      if (p.key_mask)
        window_attn_kernel<2, true><<<grid, 64 * kPromptWaves, 0, stream>>>(p);
      else
        window_attn_kernel<2, false><<<grid, 64 * kPromptWaves, 0, stream>>>(p);
    }
  } else {
    const long need = window_workspace(p);
    IRIS_REQUIRE(need == 0 || (args->workspace && aligned(args->workspace, 16) && args->workspace_bytes >= need),
                 "window_attn: needs %ld bytes of 16-byte aligned workspace", need);
    p.part_o = static_cast<float*>(args->workspace);
    p.part_ml = p.part_o + rows * p.splits * kHd;
    const long total = static_cast<long>(p.batch) * p.kv_heads * p.row_tiles * p.splits;
    IRIS_REQUIRE(total < (1L << 23), "window_attn: too many items and K/V heads");
    p.total_wg = static_cast<int>(total);
    if (p.key_mask)
      window_few_kernel<true><<<dim3(p.total_wg), 64 * kFewWaves, 0, stream>>>(p);
    else
      window_few_kernel<false><<<dim3(p.total_wg), 64 * kFewWaves, 0, stream>>>(p);
    if (p.splits > 1) window_join_kernel<<<dim3(static_cast<unsigned>((rows + 3) / 4)), 256, 0, stream>>>(p, rows);
  }
  return check_launch("window_attn");
}
