// Drawing the next token: temperature, top-k, top-p and min-p from a given uniform number per row.
//
// With m = max x and w_i = exp((x_i - m) / T), per row:
//   top-k  keeps the k largest x (equal values: lowest index first)
//   top-p  of those, in that order, the shortest prefix whose weight reaches top_p of theirs
//   min-p  of those, the ones with w_i >= min_p
// and the token is the first index i with sum_{j <= i, kept} w_j > u * sum_kept w.
//
// Which token that is must not hang on the order of a sum: weights are formed in double and rounded to
// integer multiples of 2^-42, so every sum is exact, whatever order and however many CTAs form it.
//
// One cluster of 1, 2, 4 or 8 CTAs per row; each CTA keeps its slab of the row in shared memory as
// order-preserving 32-bit keys, so HBM sees a row once and every later pass runs on chip.
#include "../../include/munet_b200.h"
#include "common.h"
#include "ptx.cuh"
#include <climits>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace mu {

constexpr int SP_THREADS = 1024, SP_WARPS = SP_THREADS / 32, SP_MAX_CLUSTER = 8;
constexpr int SP_SMEM_KEYS = 49152; // keys of one CTA that fit its shared memory (192 KB)
constexpr double SP_ONE = 4398046511104.0; // 2^42: the weight of the row's maximum

struct SampleArgs {
  const void *x;
  long long ld;
  const float *u, *temperature;
  const int *top_k;
  const float *top_p, *min_p;
  int *idx;
  float *prob;
  int cols, per_cta, in_smem;
};

constexpr uint32_t KEY_NEG_INF = 0x007fffffu, KEY_POS_INF = 0xff800000u;
// Order-preserving image of a float; NaN counts as -inf, -0 as +0.
__device__ __forceinline__ uint32_t to_key(float v) {
  if (v != v)
    return KEY_NEG_INF;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <typename T> __device__ __forceinline__ float load_logit(const T *p, long long i);
template <> __device__ __forceinline__ float load_logit<float>(const float *p, long long i) { return p[i]; }
template <> __device__ __forceinline__ float load_logit<__nv_bfloat16>(const __nv_bfloat16 *p, long long i) {
  return __bfloat162float(p[i]);
}

using u64 = unsigned long long;

struct SampleShared {
  uint32_t cnt[2][256], lo[2][256], hi[2][256]; // digit histograms: elements, weight (low and high word)
  u64 warp_sum[SP_WARPS];
  u64 total[2]; // this CTA's sum, read by the cluster
  uint32_t warp_max[SP_WARPS];
  uint32_t cta_max;
  u64 found_above;
  uint32_t found_digit, found_count;
  int found_index;
};

// Inclusive scan of v over the CTA's threads; returns this thread's, and the CTA's total in `all`.
__device__ __forceinline__ u64 block_scan(u64 v, SampleShared &sh, u64 &all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 t = __shfl_up_sync(~0u, v, d);
    if (lane >= d)
      v += t;
  }
  __syncthreads(); // warp_sum may still be read
  if (lane == 31)
    sh.warp_sum[warp] = v;
  __syncthreads();
  u64 w = sh.warp_sum[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 t = __shfl_up_sync(~0u, w, d);
    if (lane >= d)
      w += t;
  }
  all = __shfl_sync(~0u, w, 31);
  const u64 before = __shfl_sync(~0u, w, (warp + 31) & 31);
  return v + (warp ? before : 0);
}

struct Row {
  double xmax, inv_t;
  uint32_t max_key;
  bool spike; // the maximum is +inf: only elements equal to it weigh anything
  __device__ __forceinline__ double weight(uint32_t key) const {
    if (key == max_key)
      return 1.0;
    if (spike || key <= KEY_NEG_INF)
      return 0.0;
    return exp((static_cast<double>(from_key(key)) - xmax) * inv_t);
  }
  __device__ __forceinline__ u64 fixed(uint32_t key) const { return __double2ull_rn(weight(key) * SP_ONE); }
};

template <typename T> __global__ void __launch_bounds__(SP_THREADS) sample_kernel(SampleArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ SampleShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *x = static_cast<const T *>(a.x) + row * a.ld;
  const int s0 = min(rank * a.per_cta, a.cols), n = min(a.per_cta, a.cols - s0);
  x += s0;
  for (int i = tid; i < 256; i += SP_THREADS)
#pragma unroll
    for (int b = 0; b < 2; ++b)
      sh.cnt[b][i] = sh.lo[b][i] = sh.hi[b][i] = 0;

  uint32_t top = 0;
  for (int i = tid; i < n; i += SP_THREADS) {
    const uint32_t k = to_key(load_logit(x, i));
    if (a.in_smem)
      keys[i] = k;
    top = max(top, k);
  }
  top = __reduce_max_sync(~0u, top);
  if (lane == 0)
    sh.warp_max[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = __reduce_max_sync(~0u, sh.warp_max[lane]);
    if (lane == 0)
      sh.cta_max = top;
  }
  cluster.sync();
  top = 0;
  for (int r = 0; r < C; ++r)
    top = max(top, *cluster.map_shared_rank(&sh.cta_max, r));

  auto key_at = [&](int i) -> uint32_t { return a.in_smem ? keys[i] : to_key(load_logit(x, i)); };
  // a thread owns consecutive indices, an odd number of them: index order without bank conflicts
  const int per = ((n + SP_THREADS - 1) / SP_THREADS) | 1;
  const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
  int total_turn = 0, hist_turn = 0; // which of the two copies the next exchange uses

  // Index (in the row) of the t-th element, t >= 1, that equals `key`, in index order.
  auto nth_equal = [&](uint32_t key, u64 t) {
    u64 c = 0, all;
    for (int i = i0; i < i1; ++i)
      c += key_at(i) == key;
    u64 inc = block_scan(c, sh, all);
    if (tid == 0)
      sh.total[total_turn] = all, sh.found_index = -1;
    cluster.sync();
    for (int r = 0; r < rank; ++r)
      inc += *cluster.map_shared_rank(&sh.total[total_turn], r);
    total_turn ^= 1;
    if (inc >= t && inc - c < t) {
      u64 at = inc - c;
      for (int i = i0; i < i1; ++i)
        if (key_at(i) == key && ++at == t)
          for (int r = 0; r < C; ++r)
            *cluster.map_shared_rank(&sh.found_index, r) = s0 + i;
    }
    cluster.sync();
    return sh.found_index;
  };

  const float T_row = a.temperature ? a.temperature[row] : 1.f;
  if (top <= KEY_NEG_INF) { // nothing to draw from
    if (rank == 0 && tid == 0) {
      a.idx[row] = -1;
      if (a.prob)
        a.prob[row] = 0.f;
    }
  } else if (!(T_row > 0.f)) { // greedy
    const int i = nth_equal(top, 1);
    if (rank == 0 && tid == 0) {
      a.idx[row] = i;
      if (a.prob)
        a.prob[row] = 1.f;
    }
  } else {
    Row rw;
    rw.max_key = top, rw.spike = top == KEY_POS_INF;
    rw.xmax = from_key(top), rw.inv_t = 1.0 / static_cast<double>(T_row);
    // kept: key > bound_key, or equal to it at an index up to bound_idx
    uint32_t bound_key = 0;
    int bound_idx = INT_MAX;
    auto kept = [&](uint32_t k, int i) { return k > bound_key || (k == bound_key && s0 + i <= bound_idx); };

    // Of the kept elements in descending order: keep those before which less than `target` of the
    // measure (elements, or weight) lies. Eight bits of the key at a time, from the top.
    auto cut = [&](u64 target, bool by_weight) {
      u64 above = 0;
      uint32_t prefix = 0, ties = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = i0; i < i1; ++i) {
          const uint32_t k = key_at(i);
          if ((shift < 24 && (k >> (shift + 8)) != prefix) || !kept(k, i))
            continue;
          const uint32_t d = (k >> shift) & 255u;
          atomicAdd(&sh.cnt[hist_turn][d], 1u);
          if (by_weight) {
            const u64 w = rw.fixed(k);
            const uint32_t wl = static_cast<uint32_t>(w), old = atomicAdd(&sh.lo[hist_turn][d], wl);
            const uint32_t wh = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
            if (wh)
              atomicAdd(&sh.hi[hist_turn][d], wh);
          }
        }
        cluster.sync();
        if (warp == 0) { // lane l: digits 255 - 8l ... 248 - 8l
          u64 v[8], sum = 0;
          uint32_t c[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int d = 255 - 8 * lane - j;
            v[j] = 0, c[j] = 0;
            for (int r = 0; r < C; ++r) {
              c[j] += *cluster.map_shared_rank(&sh.cnt[hist_turn][d], r);
              if (by_weight)
                v[j] += (static_cast<u64>(*cluster.map_shared_rank(&sh.hi[hist_turn][d], r)) << 32) +
                        *cluster.map_shared_rank(&sh.lo[hist_turn][d], r);
            }
            if (!by_weight)
              v[j] = c[j];
            sum += v[j];
          }
          u64 inc = sum;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const u64 t = __shfl_up_sync(~0u, inc, d);
            if (lane >= d)
              inc += t;
          }
          u64 at = above + inc - sum;
          if (at < target && at + sum >= target) {
            for (int j = 0; j < 8; ++j) {
              if (at + v[j] >= target) {
                sh.found_above = at, sh.found_digit = 255 - 8 * lane - j, sh.found_count = c[j];
                break;
              }
              at += v[j];
            }
          }
        }
        __syncthreads();
        above = sh.found_above, ties = sh.found_count;
        prefix = (prefix << 8) | sh.found_digit;
        hist_turn ^= 1;
        // Whoever passed this turn's cluster.sync() has read the copy of the turn before: it is free.
        for (int i = tid; i < 256; i += SP_THREADS)
          sh.cnt[hist_turn][i] = sh.lo[hist_turn][i] = sh.hi[hist_turn][i] = 0;
        __syncthreads();
      }
      u64 t = target - above;
      if (by_weight) {
        const u64 w = rw.fixed(prefix);
        t = (t + w - 1) / w;
      }
      const int at = t < ties ? nth_equal(prefix, t) : bound_key == prefix ? bound_idx : INT_MAX;
      bound_key = prefix, bound_idx = at;
    };
    auto weight_of_kept = [&](double floor_w, u64 &mine, u64 &before) { // sum over the row
      mine = 0;
      u64 all;
      for (int i = i0; i < i1; ++i) {
        const uint32_t k = key_at(i);
        if (kept(k, i)) {
          const double w = rw.weight(k);
          if (w >= floor_w)
            mine += __double2ull_rn(w * SP_ONE);
        }
      }
      before = block_scan(mine, sh, all) - mine;
      if (tid == 0)
        sh.total[total_turn] = all;
      cluster.sync();
      u64 sum = 0;
      for (int r = 0; r < C; ++r) {
        const u64 t = *cluster.map_shared_rank(&sh.total[total_turn], r);
        if (r < rank)
          before += t;
        sum += t;
      }
      total_turn ^= 1;
      return sum;
    };

    const int k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < a.cols)
      cut(k, false);
    u64 mine, before;
    const float p = a.top_p ? a.top_p[row] : 1.f;
    if (p < 1.f) {
      const u64 all = weight_of_kept(0.0, mine, before);
      const double target = ceil(static_cast<double>(p) * static_cast<double>(all));
      cut(target >= 1.0 ? static_cast<u64>(target) : 1ull, true);
    }
    const float mp = a.min_p ? a.min_p[row] : 0.f;
    const u64 all = weight_of_kept(mp > 0.f ? fmin(static_cast<double>(mp), 1.0) : 0.0, mine, before);
    const float u = a.u[row];
    double at = u > 0.f ? static_cast<double>(u) * static_cast<double>(all) : 0.0;
    const u64 want = at >= static_cast<double>(all) ? all - 1 : static_cast<u64>(at);
    if (before <= want && want < before + mine) {
      const double floor_w = mp > 0.f ? fmin(static_cast<double>(mp), 1.0) : 0.0;
      u64 c = before;
      for (int i = i0; i < i1; ++i) {
        const uint32_t key = key_at(i);
        if (!kept(key, i))
          continue;
        const double w = rw.weight(key);
        if (w < floor_w)
          continue;
        c += __double2ull_rn(w * SP_ONE);
        if (c > want) {
          a.idx[row] = s0 + i;
          if (a.prob)
            a.prob[row] = static_cast<float>(w * SP_ONE / static_cast<double>(all));
          break;
        }
      }
    }
  }
  cluster.sync(); // nobody leaves while its shared memory may be read
}

// 0 ok, 1 dtype not implemented, 2 CUDA error
template <typename T> int launch_sample_t(SampleArgs a, int rows, int num_sms, cudaStream_t st) {
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * SP_SMEM_KEYS) !=
        cudaSuccess)
      return 2;
    once.set(1);
  }
  // As few CTAs per row as hold it in shared memory; more while the rows alone would leave SMs idle
  // and a CTA still has a few keys per thread.
  int C = 1;
  while (C < SP_MAX_CLUSTER &&
         ((a.cols + C - 1) / C > SP_SMEM_KEYS || (1ll * rows * C * 2 <= num_sms && a.cols / C > 4 * SP_THREADS)))
    C *= 2;
  a.per_cta = ((a.cols + C - 1) / C + 7) & ~7;
  a.in_smem = a.per_cta <= SP_SMEM_KEYS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * C), cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = a.in_smem ? 4ull * a.per_cta : 0, cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a) == cudaSuccess ? 0 : 2;
}
int launch_sample(const SampleArgs &a, int rows, int dtype, int num_sms, cudaStream_t st) {
  if (dtype == F32)
    return launch_sample_t<float>(a, rows, num_sms, st);
  if (dtype == BF16)
    return launch_sample_t<__nv_bfloat16>(a, rows, num_sms, st);
  return 1;
}

} // namespace mu

extern "C" {

int mu_set_error(mu_ctx *ctx, int code, const char *msg);
int mu_ctx_select_device(mu_ctx *ctx);
int mu_ctx_num_sms(const mu_ctx *ctx);

int mu_sample(mu_ctx *ctx, const void *logits, long long ld, const float *uniform, const float *temperature,
              const int32_t *top_k, const float *top_p, const float *min_p, int32_t *idx, float *prob, int rows,
              int cols, int dtype, void *stream) {
  if (!ctx)
    return MU_ERR_INVALID;
  if (rows < 0 || cols <= 0 || ld < cols)
    return mu_set_error(ctx, MU_ERR_INVALID, "sample: bad shape");
  if (cols > MU_SAMPLE_MAX_COLS || rows > (1 << 24))
    return mu_set_error(ctx, MU_ERR_SIZE, "sample: at most MU_SAMPLE_MAX_COLS columns and 2^24 rows");
  if (dtype != MU_F32 && dtype != MU_BF16)
    return mu_set_error(ctx, MU_ERR_UNSUPPORTED, "sample: dtype not implemented (float32, bfloat16)");
  if (rows == 0)
    return MU_OK;
  if (!logits || !uniform || !idx)
    return mu_set_error(ctx, MU_ERR_INVALID, "sample: null pointer");
  if (mu_ctx_select_device(ctx) != MU_OK)
    return mu_set_error(ctx, MU_ERR_CUDA, "sample: cannot select device");
  const mu::SampleArgs a{logits, ld, uniform, temperature, top_k, top_p, min_p, idx, prob, cols, 0, 0};
  if (mu::launch_sample(a, rows, dtype, mu_ctx_num_sms(ctx), static_cast<cudaStream_t>(stream)))
    return mu_set_error(ctx, MU_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
  return MU_OK;
}

} // extern "C"
