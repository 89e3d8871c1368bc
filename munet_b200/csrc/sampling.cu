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
//
// Where a cut falls is found in two steps: a histogram over 4096 buckets of the logits (1/64 or 1/128
// of a factor of two wide, from the maximum down: a monotone function, so buckets are ranges of the order) says
// in which bucket, and that bucket's few elements are sorted. With a top-k of a few hundred at most everything
// down to the cut goes into the list, which then settles top-p, min-p and the draw as well; a larger one is cut
// by its bucket alone, and top-p then goes through the kept elements' buckets. Rows whose bucket holds more than
// a list (ties, logits of another scale) are cut eight bits of the key at a time.
//
// A small batch is latency: one row of 32000 bfloat16 logits with top-k 50 takes 12 us over six cluster barriers.
// A large one is bound by the instructions of the exact weights, formed twice, and by barriers: 256 rows of 100003
// float32 logits with top-p 0.97 take 258 us (102 MB), 200 rows in bfloat16 with neither top-k nor top-p 94 us.
#include "../../include/munet_b200.h"
#include "common.h"
#include "ptx.cuh"
#include <cfloat>
#include <climits>
#include <type_traits>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace mu {

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_MAX_CLUSTER = 8;
constexpr int SP_BUCKETS = 4096, SP_LIST = 512, SP_RANKED = 256;
// 64 to a factor of two where elements are counted (44 nats of the logits themselves), 128 where weights are summed
// (a cut more than 2^32 below the maximum is rare): half the list to sort, 273 -> 265 us for 256 rows of 100003
constexpr float SP_BUCKETS_PER_NAT = 92.3325f;
constexpr int SP_TABLE_BITS = 7, SP_TABLE = 1 << SP_TABLE_BITS;
constexpr int SP_SMEM_KEYS = 43008; // keys of one CTA that fit its shared memory beside the buckets (168 KB)
constexpr int SP_PAIR_KEYS = 15360; // and of one of two CTAs of an SM: one loads while the other computes
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

constexpr uint32_t KEY_NEG_INF = 0x007fffffu;
// Order-preserving image of a float; NaN counts as -inf, -0 as +0.
__device__ __forceinline__ uint32_t to_key(float v) {
  if (v != v)
    return KEY_NEG_INF;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_key(uint32_t k) {
  return __uint_as_float(k ^ (~static_cast<uint32_t>(static_cast<int>(k) >> 31) | 0x80000000u));
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
  double table[SP_TABLE]; // 2^(i/128)
  u64 list[SP_LIST];  // (key, ~index), rank 0's
  int ranks[SP_RANKED];
  int n_list;
  int bucket;         // that the cut falls into
  u64 above, within;  // measure before it, and of it
  uint32_t bound_key; // broadcast by rank 0
  int bound_idx;
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
  u64 w = lane < SP_WARPS ? sh.warp_sum[lane] : 0;
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

// exp((x - max) / T) = 2^t, t = i/128 + f: the table's 2^(i/128) times the Taylor polynomial of 2^f up to f^4,
// |f| <= 1/256: the remainder is below (ln2/256)^5 / 120 = 1.3e-15, a hundredth of the 2^-43 that rounding to
// whole multiples of 2^-42 allows for weights near one. exp() cost twice as much.
struct Row {
  double max, c; // t = (x - max) * c, exactly 0 for the maximum
  const double *table;
  uint32_t floor_key; // below it t is under -64 (the weight under 2^-43), or there is no t: -inf, and next to a
                      // maximum of +inf everything else
  // No branches, so that several run at a time.
  __device__ __forceinline__ double weight(uint32_t key) const {
    const double d = static_cast<double>(fminf(from_key(key), FLT_MAX)) - max;
    const double shift = 0x1.8p52 / SP_TABLE; // adding it rounds to a multiple of 1/128
    const double r = fma(d, c, shift);
    const int i = __double2loint(r);
    const double f = fma(d, c, shift - r);
    double p = fma(f, 0x1.3b2ab6fba4e77p-7, 0x1.c6b08d704a0c0p-5); // ln2^k / k!
    p = fma(f, p, 0x1.ebfbdff82c58fp-3);
    p = fma(f, p, 0x1.62e42fefa39efp-1);
    p = fma(f, p, 1.0) * table[i & (SP_TABLE - 1)];
    const double w = __hiloint2double(__double2hiint(p) + ((i >> SP_TABLE_BITS) << 20), __double2loint(p));
    return key >= floor_key ? w : 0.0;
  }
  // rounded to a multiple of 2^-42, as that multiple
  __device__ __forceinline__ static u64 whole(double w) {
    return static_cast<u64>(__double_as_longlong(fma(w, SP_ONE, 0x1p52))) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 fixed(uint32_t key) const { return whole(weight(key)); }
};

// Sorts v[0 .. n) in descending order; n a power of two up to SP_THREADS, non-zero values distinct. Short lists
// by counting what is larger than each (all threads share that, three barriers); others in runs of 32 within a warp's
// registers, then run by run: an element goes where its place in its own run and that in the other say.
__device__ __forceinline__ void sort_desc(u64 *v, int *ranks, int n) {
  const int i = threadIdx.x;
  __syncthreads();
  if (n <= SP_RANKED) {
    const int e = i & (n - 1), share = max(1, n * n / SP_THREADS), from = i / n * share;
    const u64 x = v[e];
    if (i < n)
      ranks[i] = 0;
    __syncthreads();
    if (from < n) {
      int larger = 0;
#pragma unroll 8
      for (int j = from; j < from + share; ++j)
        larger += v[j] > x;
      if (larger)
        atomicAdd(&ranks[e], larger);
    }
    __syncthreads();
    if (i < n)
      v[i] = 0;
    const int at = i < n ? ranks[i] : 0;
    __syncthreads();
    if (i < n && x)
      v[at] = x;
  } else {
    u64 x = i < n ? v[i] : 0;
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) {
        const u64 y = __shfl_xor_sync(~0u, x, j);
        x = ((i & j) == 0) == ((i & k & 31) == 0) ? max(x, y) : min(x, y);
      }
    if (i < n)
      v[i] = x;
#pragma unroll 1
    for (int length = 32; length < n; length <<= 1) {
      __syncthreads();
      int at = i & (length - 1);
      x = i < n ? v[i] : 0;
      if (i < n) { // how many of the other run come first: with equal ones (zeros) the first run's do
        const bool second = i & length;
        const u64 *other = v + ((i & -length) ^ length);
        int lo = 0;
#pragma unroll 1
        for (int step = length; step > 0; step >>= 1)
          if (lo + step <= length && (second ? other[lo + step - 1] >= x : other[lo + step - 1] > x))
            lo += step;
        at += lo + (i & -(2 * length));
      }
      __syncthreads();
      if (i < n)
        v[at] = x;
    }
  }
  __syncthreads();
}

template <typename T> __global__ void __launch_bounds__(SP_THREADS, 2) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint32_t buckets[]; // [2][SP_BUCKETS], then the keys
  uint32_t *const keys = buckets + 2 * SP_BUCKETS;
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

  for (int i = tid; i < 2 * SP_BUCKETS / 4; i += SP_THREADS)
    reinterpret_cast<uint4 *>(buckets)[i] = make_uint4(0, 0, 0, 0);
  if (tid < SP_TABLE)
    sh.table[tid] = exp2(static_cast<double>(tid) / SP_TABLE);
  if (tid == 0)
    sh.n_list = 0;

  uint32_t top = 0;
  {
    auto take = [&](int i, uint32_t k) {
      if (a.in_smem)
        keys[i] = k;
      top = max(top, k);
    };
    // 16 bytes a thread from the first 16-byte boundary on, several loads in flight; the ends one by one
    constexpr int E = 16 / sizeof(T), U = 4;
    const int head = min(n, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
    const int packs = (n - head) / E;
    const uint4 *body = reinterpret_cast<const uint4 *>(x + head);
    for (int q0 = tid; q0 < packs; q0 += U * SP_THREADS) {
      uint4 v[U];
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (q0 + e * SP_THREADS < packs)
          v[e] = __ldcs(body + q0 + e * SP_THREADS);
#pragma unroll
      for (int e = 0; e < U; ++e)
        if (const int q = q0 + e * SP_THREADS; q < packs) {
          const uint32_t w[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
              take(head + 4 * q + j, to_key(__uint_as_float(w[j])));
            } else {
              take(head + 8 * q + 2 * j, to_key(bf16_lo(w[j])));
              take(head + 8 * q + 2 * j + 1, to_key(bf16_hi(w[j])));
            }
          }
        }
    }
    const int rest = n - head - packs * E; // fewer than E on either side
    if (tid < head)
      take(tid, to_key(load_logit(x, tid)));
    if (tid < rest)
      take(n - rest + tid, to_key(load_logit(x, n - rest + tid)));
  }
  top = __reduce_max_sync(~0u, top);
  if (lane == 0)
    sh.warp_max[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = __reduce_max_sync(~0u, lane < SP_WARPS ? sh.warp_max[lane] : 0u);
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
    const float xmax = from_key(top);
    rw.table = sh.table;
    rw.max = static_cast<double>(fminf(xmax, FLT_MAX)), rw.c = 1.4426950408889634 / static_cast<double>(T_row);
    // rounded to a float, which moves t by no more than from -64 to -128
    rw.floor_key = xmax > FLT_MAX ? top
                                  : max(to_key(static_cast<float>(rw.max - 44.3614195558365 * static_cast<double>(T_row))),
                                        KEY_NEG_INF + 1);
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
    auto row_sum = [&](u64 mine, u64 &before) { // over the row, and over the threads before this one
      u64 all;
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
    auto weight_of_kept = [&](double floor_w, u64 &mine, u64 &before) {
      mine = 0;
#pragma unroll 4
      for (int i = i0; i < i1; ++i) {
        const uint32_t k = key_at(i);
        const double w = rw.weight(k);
        mine += kept(k, i) && w >= floor_w ? Row::whole(w) : 0;
      }
      return row_sum(mine, before);
    };

    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f;
    const bool by_count = k > 0 && k < a.cols;
    float per_unit = by_count ? SP_BUCKETS_PER_NAT : 2.f * SP_BUCKETS_PER_NAT / T_row;
    auto bucket_of = [&](uint32_t key) { return min(SP_BUCKETS - 1, static_cast<int>((xmax - from_key(key)) * per_unit)); };
    // Fills the buckets and finds the one in which the measure (elements, or weight) reaches the target,
    // which `target_of` gives from the row's total.
    // `filtered`: kept elements only.
    auto find_bucket = [&](bool weight, auto filtered, auto target_of) {
      // Four keys and weights at a time before the first addition: to the compiler an atomic may change the keys.
      constexpr int U = 4;
      for (int i = tid; i < n; i += U * SP_THREADS) {
        uint32_t key[U];
        u64 w[U];
#pragma unroll
        for (int e = 0; e < U; ++e)
          key[e] = i + e * SP_THREADS < n ? key_at(i + e * SP_THREADS) : KEY_NEG_INF;
#pragma unroll
        for (int e = 0; e < U; ++e)
          w[e] = weight && (!decltype(filtered)::value || kept(key[e], i + e * SP_THREADS)) ? rw.fixed(key[e]) : 0;
#pragma unroll
        for (int e = 0; e < U; ++e) {
          const int b = bucket_of(key[e]);
          if (!weight) {
            if (i + e * SP_THREADS < n)
              atomicAdd(&buckets[b], 1u);
          } else if (w[e]) {
            const uint32_t wl = static_cast<uint32_t>(w[e]), old = atomicAdd(&buckets[b], wl);
            const uint32_t wh = static_cast<uint32_t>(w[e] >> 32) + (old + wl < old ? 1u : 0u);
            if (wh)
              atomicAdd(&buckets[SP_BUCKETS + b], wh);
          }
        }
      }
      cluster.sync();
      // Rank r sums up the cluster's buckets [r, r + 1) * SP_BUCKETS / C; the ranks' totals say whose hold the cut.
      const int share = SP_BUCKETS / C, per_thread = (share + SP_THREADS - 1) / SP_THREADS; // 1 .. 8
      const int b0 = rank * share + tid * per_thread;
      u64 v[SP_BUCKETS / SP_THREADS], sum = 0, all;
#pragma unroll
      for (int j = 0; j < SP_BUCKETS / SP_THREADS; ++j) {
        v[j] = 0;
        if (j < per_thread && tid * per_thread + j < share) {
          uint32_t lo[SP_MAX_CLUSTER], hi[SP_MAX_CLUSTER]; // all remote loads before the first sum
#pragma unroll
          for (int r = 0; r < SP_MAX_CLUSTER; ++r) {
            lo[r] = hi[r] = 0;
            if (r < C) {
              const uint32_t *from = cluster.map_shared_rank(buckets, r) + b0 + j;
              lo[r] = from[0];
              if (weight)
                hi[r] = from[SP_BUCKETS];
            }
          }
#pragma unroll
          for (int r = 0; r < SP_MAX_CLUSTER; ++r)
            v[j] += lo[r] + (static_cast<u64>(hi[r]) << 32);
        }
        sum += v[j];
      }
      u64 at = block_scan(sum, sh, all) - sum;
      if (tid == 0)
        sh.total[total_turn] = all;
      cluster.sync();
      u64 whole = 0, lower = 0;
      for (int r = 0; r < C; ++r) {
        const u64 t = *cluster.map_shared_rank(&sh.total[total_turn], r);
        whole += t;
        if (r < rank)
          lower += t;
      }
      total_turn ^= 1;
      at += lower;
      const u64 target = target_of(whole);
      if (at < target && at + sum >= target) {
        int j = 0;
        u64 within = 0;
#pragma unroll
        for (int e = 0; e < SP_BUCKETS / SP_THREADS; ++e)
          if (e == j) {
            within = v[e];
            if (at + within < target)
              at += within, ++j;
          }
        for (int r = 0; r < C; ++r) {
          SampleShared &o = *cluster.map_shared_rank(&sh, r);
          o.bucket = b0 + j, o.above = at, o.within = within;
        }
      }
      cluster.sync();
      return target;
    };
    auto to_list = [&](uint32_t key, int i) { // rank 0's
      const int at = atomicAdd(cluster.map_shared_rank(&sh.n_list, 0), 1);
      if (at < SP_LIST)
        cluster.map_shared_rank(sh.list, 0)[at] = static_cast<u64>(key) << 32 | static_cast<uint32_t>(~(s0 + i));
    };
    auto list_length = [&] {
      cluster.sync();
      return *cluster.map_shared_rank(&sh.n_list, 0);
    };
    // Puts the elements of buckets first .. last into the list; their number over the row.
    auto gather = [&](int first, int last) {
      constexpr int U = 8;
      for (int i = tid; i < n; i += U * SP_THREADS) {
        uint32_t key[U];
#pragma unroll
        for (int e = 0; e < U; ++e)
          key[e] = i + e * SP_THREADS < n ? key_at(i + e * SP_THREADS) : 0;
#pragma unroll
        for (int e = 0; e < U; ++e)
          if (const int b = bucket_of(key[e]); i + e * SP_THREADS < n && b >= first && b <= last)
            to_list(key[e], i + e * SP_THREADS);
      }
      return list_length();
    };
    // rank 0: the list in descending order (largest key, then lowest index), one element to a thread
    auto sorted = [&](int count) {
      int m = 1;
      while (m < count)
        m <<= 1;
      if (tid >= count && tid < m)
        sh.list[tid] = 0;
      sort_desc(sh.list, sh.ranks, m);
      return tid < count ? sh.list[tid] : 0ull;
    };
    // The bound: of the list's elements the last one before which less than the target lies.
    auto bound_in_list = [&](int count, u64 above, u64 target, bool weight) {
      if (rank == 0) {
        const u64 e = sorted(count);
        const u64 w = tid >= count ? 0 : weight ? rw.fixed(static_cast<uint32_t>(e >> 32)) : 1;
        u64 sum;
        const u64 ahead = above + block_scan(w, sh, sum) - w;
        if (tid < count && ahead < target && (ahead + w >= target || tid == count - 1))
          for (int r = 0; r < C; ++r) {
            *cluster.map_shared_rank(&sh.bound_key, r) = static_cast<uint32_t>(e >> 32);
            *cluster.map_shared_rank(&sh.bound_idx, r) = static_cast<int>(~static_cast<uint32_t>(e));
          }
      }
      cluster.sync();
      bound_key = sh.bound_key, bound_idx = sh.bound_idx;
    };
    const float mp = a.min_p && a.min_p[row] > 0.f ? fminf(a.min_p[row], 1.f) : 0.f;
    const float u = a.u[row];
    auto draw = [&](u64 all) { // the whole weight that lies before the drawn token's end
      const double at = u > 0.f ? static_cast<double>(u) * static_cast<double>(all) : 0.0;
      return at >= static_cast<double>(all) ? all - 1 : static_cast<u64>(at);
    };
    auto share_of = [&](u64 all) { // top_p of a sum, rounded up
      const double t = ceil(static_cast<double>(p) * static_cast<double>(all));
      return t >= 1.0 ? static_cast<u64>(t) : 1ull;
    };

    if (by_count) {
      find_bucket(false, std::false_type{}, [&](u64) { return static_cast<u64>(k); });
      const int last = sh.bucket;
      // elements down to the cut's bucket: the list has room, or nobody gathers
      const int count = sh.above + sh.within <= SP_LIST ? gather(0, last) : SP_LIST + 1;
      if (count <= SP_LIST) {
        if (rank == 0) {
          const u64 e = sorted(count);
          const uint32_t key = static_cast<uint32_t>(e >> 32);
          const double w = rw.weight(key);
          bool in = tid < min(k, count);
          u64 all;
          if (p < 1.f) {
            const u64 mine = in ? Row::whole(w) : 0, before = block_scan(mine, sh, all) - mine;
            in = in && before < share_of(all);
          }
          in = in && (!(mp > 0.f) || w >= mp);
          // in index order: sort by ~index, descending; the position rides along
          __syncthreads();
          int m = 1;
          while (m < count)
            m <<= 1;
          if (tid < m)
            sh.list[tid] = in ? (e << 32) | key : 0ull;
          sort_desc(sh.list, sh.ranks, m);
          const u64 f = tid < m ? sh.list[tid] : 0ull;
          const uint32_t fk = static_cast<uint32_t>(f);
          const double fw = f ? rw.weight(fk) : 0.0;
          const u64 mine = f ? Row::whole(fw) : 0, upto = block_scan(mine, sh, all);
          const u64 want = draw(all);
          if (upto - mine <= want && want < upto) {
            a.idx[row] = static_cast<int>(~static_cast<uint32_t>(f >> 32));
            if (a.prob)
              a.prob[row] = static_cast<float>(fw * SP_ONE / static_cast<double>(all));
          }
        }
        cluster.sync();
        return;
      }
      if (sh.within <= SP_LIST) // a large k: the cut's bucket alone
        bound_in_list(gather(last, last), sh.above, k, false);
      else
        cut(k, false);
      // Everybody has passed a cluster.sync() since reading them: buckets and list start afresh for top-p.
      if (p < 1.f) {
        for (int i = tid; i < 2 * SP_BUCKETS / 4; i += SP_THREADS)
          reinterpret_cast<uint4 *>(buckets)[i] = make_uint4(0, 0, 0, 0);
        if (tid == 0)
          sh.n_list = 0;
        per_unit = 2.f * SP_BUCKETS_PER_NAT / T_row;
        __syncthreads();
      }
    }
    const double floor_w = mp > 0.f ? static_cast<double>(mp) : 0.0;
    u64 mine = 0, before, all = 0;
    bool summed = false;
    auto top_p = [&](auto filtered) {
      const u64 target = find_bucket(true, filtered, share_of);
      const int last = sh.bucket;
      const u64 above = sh.above;
      // One pass sums up what lies above the cut's bucket and puts that bucket's elements into the list;
      // which of those are kept is added when the list is sorted. Bit b: some element i0 + b + 64 m is one.
      u64 open = 0;
#pragma unroll 4
      for (int i = i0; i < i1; ++i) {
        const uint32_t key = key_at(i);
        const int b = bucket_of(key);
        const double w = rw.weight(key);
        const bool in = !decltype(filtered)::value || kept(key, i);
        mine += in && b < last && w >= floor_w ? Row::whole(w) : 0;
        if (in && b == last) {
          open |= 1ull << ((i - i0) & 63);
          to_list(key, i);
        }
      }
      const int count = list_length();
      if (count > SP_LIST)
        return;
      summed = true;
      bound_in_list(count, above, target, true);
      for (; open; open &= open - 1)
        for (int i = i0 + __ffsll(static_cast<long long>(open)) - 1; i < i1; i += 64) {
          const uint32_t key = key_at(i);
          const double w = rw.weight(key);
          mine += bucket_of(key) == last && kept(key, i) && w >= floor_w ? Row::whole(w) : 0;
        }
      all = row_sum(mine, before);
    };
    if (p < 1.f) {
      if (by_count)
        top_p(std::true_type{});
      else
        top_p(std::false_type{});
      if (!summed)
        cut(share_of(weight_of_kept(0.0, mine, before)), true);
    }
    if (!summed)
      all = weight_of_kept(floor_w, mine, before);
    cluster.barrier_arrive(); // what follows reads nobody else's shared memory
    const u64 want = draw(all);
    // the warp of the thread whose elements hold the drawn one walks through them
    const unsigned who = __ballot_sync(~0u, before <= want && want < before + mine);
    if (who) {
      const int from = __ffs(who) - 1, j0 = __shfl_sync(~0u, i0, from), j1 = __shfl_sync(~0u, i1, from);
      u64 c = __shfl_sync(~0u, before, from);
      for (int j = j0; j < j1; j += 32) {
        const int i = j + lane;
        const uint32_t key = i < j1 ? key_at(i) : 0;
        const double w = i < j1 ? rw.weight(key) : 0.0;
        u64 inc = i < j1 && kept(key, i) && w >= floor_w ? Row::whole(w) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const u64 t = __shfl_up_sync(~0u, inc, d);
          if (lane >= d)
            inc += t;
        }
        const unsigned over = __ballot_sync(~0u, c + inc > want);
        if (over) {
          if (lane == __ffs(over) - 1) {
            a.idx[row] = s0 + i;
            if (a.prob)
              a.prob[row] = static_cast<float>(w * SP_ONE / static_cast<double>(all));
          }
          break;
        }
        c += __shfl_sync(~0u, inc, 31);
      }
    }
    cluster.barrier_wait();
    return;
  }
  cluster.sync(); // nobody leaves while its shared memory may be read
}

// 0 ok, 1 dtype not implemented, 2 CUDA error
template <typename T> int launch_sample_t(SampleArgs a, int rows, int num_sms, cudaStream_t st) {
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             4 * (2 * SP_BUCKETS + SP_SMEM_KEYS)) !=
        cudaSuccess)
      return 2;
    once.set(1);
  }
  // As few CTAs per row as leave room for a second one on their SM (or at least hold the row); more while the
  // rows alone would leave SMs idle and a CTA still has a few keys per thread.
  int C = 1;
  while (C < SP_MAX_CLUSTER && ((a.cols + C - 1) / C > SP_PAIR_KEYS ||
                                (1ll * rows * C <= num_sms && a.cols / C > 4 * SP_THREADS)))
    C *= 2;
  a.per_cta = ((a.cols + C - 1) / C + 7) & ~7;
  a.in_smem = a.per_cta <= SP_SMEM_KEYS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * C), cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = 4ull * (2 * SP_BUCKETS + (a.in_smem ? a.per_cta : 0)), cfg.stream = st;
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
