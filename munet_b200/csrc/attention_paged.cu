// Attention over a paged KV cache held in e4m3 with one scale per page and head (layout: kv_cache.cu).
//
//   out[t, hq, :] = sum_j softmax_j( q[t, hq, :] . K[j, hk, :] / sqrt(D) ) V[j, hk, :],  hk = hq / G
//
// Token i of a request with n new tokens and `len` tokens in the cache sits at position len - n + i;
// causal attention lets it see j <= that position. A row that sees nothing gives zeros.
//
// Work split (both kernels): a request's rows (token, head of the group) are cut into row tiles, its
// keys into chunks of 128 tokens; (request, KV head, row tile, chunk) in this order is one long list of
// units that the resident CTAs share out evenly, whatever the lengths are. A CTA walks its range as
// segments, one per (request, head, row tile). A segment that covers all chunks writes its rows; one
// that does not leaves (running maximum, sum, weighted values) in the workspace, and a second small
// kernel joins them. No atomics: results do not depend on the order in which CTAs run.
#include "../../include/munet_b200.h"
#include "common.h"
#include "ptx.cuh"
#include <climits>
#include <cmath>
#include <type_traits>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace mu {

struct PagedArgs {
  const void *q;
  void *out;
  long long q_ld, out_ld; // elements between tokens
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *table;
  int table_stride;
  const int *query_start, *seq_lens;
  int B, n_tokens, Hq, Hkv, G, D, num_pages, page_size, causal;
  float scale_log2; // log2(e) / sqrt(D)
  struct SplitItem *items;
  float2 *part_ml;
  float *part_o;
  int rows_per_tile; // stride of the partial results
  int *status;
};

// A (request, head, row tile) whose chunks went to more than one CTA; entry c belongs to the CTA that
// holds its first chunk. Its later pieces are the first segments of CTAs c+1 .. last_cta.
struct SplitItem {
  int used, first_slot, last_cta, row0, n_rows, q0, head;
};

constexpr int CHUNK = 128; // tokens per unit

struct Seq {
  int q0, nq, len;  // first row of q, new tokens, tokens in the cache (as given)
  int seen;         // tokens the block table can address
};
__device__ __forceinline__ Seq load_seq(const PagedArgs &a, int b) {
  Seq s;
  s.q0 = a.query_start[b];
  const int q1 = a.query_start[b + 1];
  s.nq = q1 - s.q0;
  s.len = a.seq_lens[b];
  if (s.q0 < 0 || q1 < s.q0 || q1 > a.n_tokens || s.len < 0) {
    atomicCAS(a.status, 0, MU_DEV_BAD_LENGTH);
    s.nq = 0, s.len = 0;
  }
  const long long room = 1ll * a.table_stride * a.page_size;
  s.seen = s.len;
  if (s.nq > 0 && s.len > room) {
    atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
    s.seen = static_cast<int>(room);
  }
  return s;
}
__device__ __forceinline__ int chunks_of(const Seq &s) { return s.seen > 0 ? (s.seen - 1) / CHUNK + 1 : 1; }
__device__ __forceinline__ long long units_of(const PagedArgs &a, const Seq &s, int R) {
  if (s.nq <= 0)
    return 0;
  const long long rows = 1ll * s.nq * a.G;
  return a.Hkv * ((rows + R - 1) / R) * chunks_of(s);
}
// Keys row `row` of a request may see.
__device__ __forceinline__ int row_limit(const PagedArgs &a, const Seq &s, long long row) {
  if (row >= 1ll * s.nq * a.G)
    return 0;
  if (!a.causal)
    return s.seen;
  const int i = static_cast<int>(row / a.G);
  return max(0, min(s.seen, s.len - s.nq + i + 1));
}

// Inclusive prefix of units over the requests into shared memory; returns the total.
template <int THREADS, int R>
__device__ __forceinline__ long long scan_units(const PagedArgs &a, long long *upto, long long *warp_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) {
    sum += units_of(a, load_seq(a, b), R);
    upto[b] = sum;
  }
  long long inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long t = __shfl_up_sync(~0u, inc, d);
    if (lane >= d)
      inc += t;
  }
  if (lane == 31)
    warp_sum[warp] = inc;
  __syncthreads();
  long long before = inc - sum, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp)
      before += warp_sum[w];
    total += warp_sum[w];
  }
  for (int b = b0; b < b1; ++b)
    upto[b] += before;
  __syncthreads();
  return total;
}

struct Segment {
  int b, head, n_rows;   // request, KV head, rows of the tile that exist
  long long row0;        // first row of the tile
  int chunk0, chunks;    // range of this CTA
  int slot;              // -1: complete
};

// Walks one CTA's share of the unit list.
struct Walk {
  long long u, end, total;
  int grid, cta, b;
  bool first;
  __device__ __forceinline__ Walk(long long total_, int cta_, int grid_) : total(total_), cta(cta_), b(0), first(true) {
    grid = static_cast<int>(min(static_cast<long long>(grid_), total_)); // every active CTA has a unit
    if (cta < grid) {
      u = total / grid * cta + total % grid * cta / grid;
      end = total / grid * (cta + 1) + total % grid * (cta + 1) / grid;
    } else {
      u = end = 0;
    }
  }
  // CTA that holds unit x: the largest c with start(c) <= x. start(c) = floor(total * c / grid).
  __device__ __forceinline__ int owner(long long x) const {
    int lo = 0, hi = grid - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (total / grid * mid + total % grid * mid / grid <= x)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  }
  template <int R>
  __device__ __forceinline__ bool next(const PagedArgs &a, const long long *upto, Segment &g, Seq &s) {
    if (u >= end)
      return false;
    int lo = b, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (upto[mid] > u)
        hi = mid;
      else
        lo = mid + 1;
    }
    b = lo;
    s = load_seq(a, b);
    const long long base = b ? upto[b - 1] : 0;
    const long long rows = 1ll * s.nq * a.G;
    const long long tiles = (rows + R - 1) / R;
    const int nc = chunks_of(s);
    const long long item = (u - base) / nc;
    g.b = b;
    g.head = static_cast<int>(item / tiles);
    g.row0 = item % tiles * R;
    g.n_rows = static_cast<int>(min(rows - g.row0, static_cast<long long>(R)));
    g.chunk0 = static_cast<int>((u - base) % nc);
    g.chunks = static_cast<int>(min(static_cast<long long>(nc - g.chunk0), end - u));
    g.slot = -1;
    if (g.chunks < nc) {
      g.slot = 2 * cta + (first ? 0 : 1);
      if (g.chunk0 == 0 && threadIdx.x == 0) {
        SplitItem it;
        it.used = 1, it.first_slot = g.slot, it.last_cta = owner(u + nc - 1);
        it.row0 = static_cast<int>(g.row0), it.n_rows = g.n_rows, it.q0 = s.q0, it.head = g.head;
        a.items[cta] = it;
      }
    }
    u += g.chunks;
    first = false;
    return true;
  }
};

__device__ __forceinline__ void store_out(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float load_in(const float *p) { return *p; }
__device__ __forceinline__ float load_in(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
// weight of a piece whose running maximum is m where the whole's is M
__device__ __forceinline__ float rel_weight(float m, float M) { return M == -INFINITY ? 1.f : ex2_approx(m - M); }

// ---- CUDA-core kernel: float32, and every head size -----------------------------------------------
// float32 queries keep float32 products and sums. Per warp a tile of 32 keys: for the scores a lane
// owns a key (its row is D consecutive bytes), for the weighted values a lane owns four dimensions.
// VB: bytes per load (16 / 4 / 1 by the head size), RT rows share every key, NA units per lane.
constexpr int SIMT_WARPS = 4, SIMT_THREADS = 32 * SIMT_WARPS;

__device__ __forceinline__ float2 fp8x2_to_float2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return __half22float2(static_cast<__half2>(h));
}

template <typename T, int RT, int VB, int NA>
__global__ void __launch_bounds__(SIMT_THREADS) attention_paged_simt_kernel(PagedArgs a) {
  constexpr int W = VB >= 4 ? 4 : 1; // dimensions of one unit
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ long long warp_sum[SIMT_WARPS];
  __shared__ float p_s[SIMT_WARPS][RT][32];
  __shared__ long long row_s[SIMT_WARPS][32];
  __shared__ float2 ml_s[SIMT_WARPS][RT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nu = a.D / W, groups = max(1, 32 / nu);
  const int unit = nu < 32 ? lane % nu : lane, group = nu < 32 ? lane / nu : 0;
  const int Dq = (a.D + 3) & ~3;
  long long *upto = reinterpret_cast<long long *>(smem_raw);
  float *q_s = reinterpret_cast<float *>(upto + ((a.B + 1) & ~1)); // [RT][Dq]
  float *o_s = q_s + RT * Dq;                                        // [warps][groups][RT][D]

  if (tid == 0)
    a.items[blockIdx.x].used = 0;
  const long long total = scan_units<SIMT_THREADS, RT>(a, upto, warp_sum);
  if (total == 0)
    return;
  Walk walk(total, blockIdx.x, gridDim.x);
  Segment g;
  Seq s;
  const unsigned ps = a.page_size;
  while (walk.next<RT>(a, upto, g, s)) {
    for (int e = tid; e < RT * Dq; e += SIMT_THREADS) {
      const int r = e / Dq, d = e - r * Dq;
      float v = 0.f;
      if (r < g.n_rows && d < a.D) {
        const long long row = g.row0 + r;
        v = load_in(static_cast<const T *>(a.q) + (s.q0 + row / a.G) * a.q_ld +
                    (1ll * g.head * a.G + row % a.G) * a.D + d);
      }
      q_s[e] = v * a.scale_log2;
    }
    __syncthreads();
    int limit[RT], least = INT_MAX, most = 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      limit[r] = row_limit(a, s, g.row0 + r);
      if (r < g.n_rows)
        least = min(least, limit[r]), most = max(most, limit[r]);
    }
    float m[RT], l[RT], acc[RT][NA][W];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
      for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int w = 0; w < W; ++w)
          acc[r][n][w] = 0.f;
    }
    for (int c = g.chunk0; c < g.chunk0 + g.chunks; ++c) {
      const int base = c * CHUNK + warp * 32;
      if (base >= most)
        break;
      const int j = base + lane;
      long long row = -1;
      float kscale = 0.f, vscale = 0.f;
      if (j < most) {
        const int page = a.table[1ll * g.b * a.table_stride + j / ps];
        if (page >= 0 && page < a.num_pages) {
          const long long tile = 1ll * page * a.Hkv + g.head;
          row = tile * ps + j % ps;
          kscale = a.ks[tile], vscale = a.vs[tile];
        } else {
          atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
        }
      }
      const bool checked = base + 32 > least || __any_sync(~0u, row < 0);
      float sc[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r)
        sc[r] = 0.f;
      if (row >= 0) {
        const uint8_t *k = a.kc + row * a.D;
        if constexpr (VB == 16) {
#pragma unroll 2
          for (int d = 0; d < a.D; d += 16) {
            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(k + d));
            const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 x = fp8x2_to_float2(w4[i] & 0xffffu), y = fp8x2_to_float2(w4[i] >> 16);
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                const float4 qv = *reinterpret_cast<const float4 *>(q_s + r * Dq + d + 4 * i);
                sc[r] = fmaf(qv.x, x.x, fmaf(qv.y, x.y, fmaf(qv.z, y.x, fmaf(qv.w, y.y, sc[r]))));
              }
            }
          }
        } else if constexpr (VB == 4) {
          for (int d = 0; d < a.D; d += 4) {
            const uint32_t w4 = __ldg(reinterpret_cast<const uint32_t *>(k + d));
            const float2 x = fp8x2_to_float2(w4 & 0xffffu), y = fp8x2_to_float2(w4 >> 16);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const float4 qv = *reinterpret_cast<const float4 *>(q_s + r * Dq + d);
              sc[r] = fmaf(qv.x, x.x, fmaf(qv.y, x.y, fmaf(qv.z, y.x, fmaf(qv.w, y.y, sc[r]))));
            }
          }
        } else {
          for (int d = 0; d < a.D; ++d) {
            const float x = fp8x2_to_float2(__ldg(k + d)).x;
#pragma unroll
            for (int r = 0; r < RT; ++r)
              sc[r] = fmaf(q_s[r * Dq + d], x, sc[r]);
          }
        }
      }
      row_s[warp][lane] = row;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const bool see = row >= 0 && j < limit[r];
        const float t = see ? sc[r] * kscale : -INFINITY;
        float top = t;
#pragma unroll
        for (int d = 16; d; d >>= 1)
          top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
        const float M = fmaxf(m[r], top), ref = M == -INFINITY ? 0.f : M;
        const float old = ex2_approx(m[r] - ref);
        const float p = see ? ex2_approx(t - ref) : 0.f;
        float sum = p;
#pragma unroll
        for (int d = 16; d; d >>= 1)
          sum += __shfl_xor_sync(~0u, sum, d);
        l[r] = l[r] * old + sum;
        m[r] = M;
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
          for (int w = 0; w < W; ++w)
            acc[r][n][w] *= old;
        // a masked key is marked, not weighted with zero: its value may be anything
        p_s[warp][r][lane] = see ? p * vscale : -1.f;
      }
      __syncwarp();
      const int count = min(32, most - base);
      auto values = [&](auto check) {
#pragma unroll 4
        for (int t = group; t < count; t += groups) {
          const long long vr = row_s[warp][t];
          if (decltype(check)::value && vr < 0)
            continue;
          const uint8_t *v = a.vc + vr * a.D;
          float x[NA][W];
#pragma unroll
          for (int n = 0; n < NA; ++n) {
            const int un = unit + 32 * n;
            const bool in = un < nu;
            if constexpr (W == 4) {
              const uint32_t w4 = in ? __ldg(reinterpret_cast<const uint32_t *>(v) + un) : 0u;
              const float2 lo = fp8x2_to_float2(w4 & 0xffffu), hi = fp8x2_to_float2(w4 >> 16);
              x[n][0] = lo.x, x[n][1] = lo.y, x[n][2] = hi.x, x[n][3] = hi.y;
            } else {
              x[n][0] = in ? fp8x2_to_float2(__ldg(v + un)).x : 0.f;
            }
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float p = p_s[warp][r][t];
            if (decltype(check)::value && p < 0.f)
              continue;
#pragma unroll
            for (int n = 0; n < NA; ++n)
#pragma unroll
              for (int w = 0; w < W; ++w)
                acc[r][n][w] = fmaf(p, x[n][w], acc[r][n][w]);
          }
        }
      };
      if (group < groups) {
        if (checked)
          values(std::true_type{});
        else
          values(std::false_type{});
      }
      __syncwarp();
    }
    // join the warps
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
        ml_s[warp][r] = make_float2(m[r], l[r]);
    }
    if (group < groups) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const int un = unit + 32 * n;
            if (un < nu)
              o_s[((warp * groups + group) * RT + r) * a.D + un * W + w] = acc[r][n][w];
          }
    }
    __syncthreads();
    for (int e = tid; e < g.n_rows * a.D; e += SIMT_THREADS) {
      const int r = e / a.D, d = e - r * a.D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < SIMT_WARPS; ++w)
        M = fmaxf(M, ml_s[w][r].x);
      float sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < SIMT_WARPS; ++w) {
        const float f = rel_weight(ml_s[w][r].x, M);
        float x = 0.f;
        for (int gi = 0; gi < groups; ++gi)
          x += o_s[((w * groups + gi) * RT + r) * a.D + d];
        sum += f * ml_s[w][r].y, o += f * x;
      }
      if (g.slot < 0) {
        const long long row = g.row0 + r;
        store_out(static_cast<T *>(a.out) + (s.q0 + row / a.G) * a.out_ld +
                      (1ll * g.head * a.G + row % a.G) * a.D + d,
                  sum == 0.f ? 0.f : o / sum);
      } else {
        const long long pr = 1ll * g.slot * a.rows_per_tile + r;
        a.part_o[pr * a.D + d] = o;
        if (d == 0)
          a.part_ml[pr] = make_float2(M, sum);
      }
    }
    __syncthreads();
  }
}

// ---- joining the pieces ---------------------------------------------------------------------------
// One CTA per (first CTA of a split item, row). Launched so that it may become resident while the main
// kernel drains; griddepcontrol.wait is what orders its reads after that kernel's writes.
constexpr int JOIN_THREADS = 128;
template <typename T> __global__ void __launch_bounds__(JOIN_THREADS) attention_paged_join_kernel(PagedArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const SplitItem it = a.items[blockIdx.x];
  const int r = blockIdx.y;
  if (!it.used || r >= it.n_rows)
    return;
  __shared__ float red[JOIN_THREADS / 32];
  const int tid = threadIdx.x, pieces = it.last_cta - static_cast<int>(blockIdx.x) + 1;
  auto slot_row = [&](int i) {
    return 1ll * (i == 0 ? it.first_slot : 2 * (static_cast<int>(blockIdx.x) + i)) * a.rows_per_tile + r;
  };
  float M = -INFINITY;
  for (int i = tid; i < pieces; i += JOIN_THREADS)
    M = fmaxf(M, a.part_ml[slot_row(i)].x);
#pragma unroll
  for (int d = 16; d; d >>= 1)
    M = fmaxf(M, __shfl_xor_sync(~0u, M, d));
  if ((tid & 31) == 0)
    red[tid >> 5] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JOIN_THREADS / 32; ++w)
    M = fmaxf(M, red[w]);
  const long long row = 1ll * it.row0 + r;
  T *out = static_cast<T *>(a.out) + (it.q0 + row / a.G) * a.out_ld + (1ll * it.head * a.G + row % a.G) * a.D;
  for (int d = tid; d < a.D; d += JOIN_THREADS) {
    float sum = 0.f, o = 0.f;
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) {
      const long long pr = slot_row(i);
      const float2 ml = a.part_ml[pr];
      const float f = rel_weight(ml.x, M);
      sum += f * ml.y, o += f * a.part_o[pr * a.D + d];
    }
    store_out(out + d, sum == 0.f ? 0.f : o / sum);
  }
}

// ---- host -----------------------------------------------------------------------------------------
constexpr int SIMT_CTAS_PER_SM = 4;
constexpr int MAX_ROWS = 16, MAX_CTAS_PER_SM = 4;

size_t paged_workspace_bytes(int num_sms, int D) {
  const size_t ctas = static_cast<size_t>(num_sms) * MAX_CTAS_PER_SM;
  return ctas * sizeof(SplitItem) + 64 + 2 * ctas * MAX_ROWS * (sizeof(float2) + sizeof(float) * D);
}

template <typename T> int launch_join(const PagedArgs &a, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, a.rows_per_tile), cfg.blockDim = dim3(JOIN_THREADS), cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attention_paged_join_kernel<T>, a) == cudaSuccess ? 0 : 2;
}

template <typename T, int RT, int VB, int NA> int launch_simt(PagedArgs a, int num_sms, cudaStream_t st) {
  constexpr int W = VB >= 4 ? 4 : 1;
  const int nu = a.D / W, groups = nu < 32 ? 32 / nu : 1, Dq = (a.D + 3) & ~3;
  const size_t smem = 8ull * ((a.B + 1) & ~1) + sizeof(float) * (RT * Dq + 1ull * SIMT_WARPS * groups * RT * a.D);
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(attention_paged_simt_kernel<T, RT, VB, NA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             200 * 1024) != cudaSuccess)
      return 2;
    once.set(1);
  }
  const int ctas = num_sms * SIMT_CTAS_PER_SM;
  a.rows_per_tile = RT;
  attention_paged_simt_kernel<T, RT, VB, NA><<<ctas, SIMT_THREADS, smem, st>>>(a);
  if (cudaGetLastError() != cudaSuccess)
    return 2;
  return launch_join<T>(a, ctas, st);
}
template <typename T, int VB, int NA> int launch_simt_rows(const PagedArgs &a, int num_sms, cudaStream_t st) {
  // rows that share a key: the group's heads for single tokens, up to 8 otherwise
  const int rows = a.n_tokens <= a.B ? a.G : 8;
  if (rows <= 1)
    return launch_simt<T, 1, VB, NA>(a, num_sms, st);
  if (rows <= 4)
    return launch_simt<T, 4, VB, NA>(a, num_sms, st);
  return launch_simt<T, 8, VB, NA>(a, num_sms, st);
}
template <typename T> int launch_simt_dim(const PagedArgs &a, int num_sms, cudaStream_t st) {
  if (a.D % 16 == 0)
    return a.D <= 128 ? launch_simt_rows<T, 16, 1>(a, num_sms, st) : launch_simt_rows<T, 16, 2>(a, num_sms, st);
  if (a.D % 4 == 0)
    return a.D <= 128 ? launch_simt_rows<T, 4, 1>(a, num_sms, st) : launch_simt_rows<T, 4, 2>(a, num_sms, st);
  return launch_simt_rows<T, 1, 8>(a, num_sms, st);
}

// 0 ok, 1 dtype not implemented, 2 CUDA error
int launch_attention_paged(PagedArgs a, void *workspace, int dtype, int num_sms, cudaStream_t st) {
  const size_t ctas = static_cast<size_t>(num_sms) * MAX_CTAS_PER_SM;
  unsigned char *w = static_cast<unsigned char *>(workspace);
  a.part_o = reinterpret_cast<float *>(w);
  w += sizeof(float) * 2 * ctas * MAX_ROWS * a.D;
  a.part_ml = reinterpret_cast<float2 *>(w);
  w += sizeof(float2) * 2 * ctas * MAX_ROWS;
  a.items = reinterpret_cast<SplitItem *>(w);
  if (dtype == F32)
    return launch_simt_dim<float>(a, num_sms, st);
  if (dtype == BF16)
    return launch_simt_dim<__nv_bfloat16>(a, num_sms, st);
  return 1;
}

} // namespace mu

extern "C" {

int mu_set_error(mu_ctx *ctx, int code, const char *msg);
int mu_ctx_select_device(mu_ctx *ctx);
int mu_ctx_num_sms(const mu_ctx *ctx);
int *mu_ctx_status_ptr(mu_ctx *ctx);

size_t mu_attention_paged_workspace_bytes(const mu_ctx *ctx, int n_tokens, int B, int Hq, int Hkv, int D, int dtype) {
  (void)dtype;
  if (!ctx || n_tokens <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0)
    return 0;
  return mu::paged_workspace_bytes(mu_ctx_num_sms(ctx), D);
}

int mu_attention_paged(mu_ctx *ctx, const void *q, long long q_ld, void *out, long long out_ld, const void *k_cache,
                       const void *v_cache, const float *k_scale, const float *v_scale, const int32_t *block_table,
                       int table_stride, const int32_t *query_start, const int32_t *seq_lens, int B, int n_tokens,
                       int Hq, int Hkv, int D, int num_pages, int page_size, int causal, int dtype, void *workspace,
                       size_t workspace_bytes, void *stream) {
  if (!ctx)
    return MU_ERR_INVALID;
  if (B < 0 || n_tokens < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || num_pages < 0 || page_size <= 0 || table_stride < 0)
    return mu_set_error(ctx, MU_ERR_INVALID, "attention_paged: bad dimensions");
  if (Hq % Hkv != 0)
    return mu_set_error(ctx, MU_ERR_INVALID, "attention_paged: query heads must be a multiple of the KV heads");
  if (page_size % 16 != 0 || page_size > 1024 || D > 256 || Hkv > 16384)
    return mu_set_error(ctx, MU_ERR_UNSUPPORTED, "attention_paged: page size a multiple of 16 up to 1024, head size "
                        "up to 256, at most 16384 heads");
  if (dtype != MU_F32 && dtype != MU_BF16)
    return mu_set_error(ctx, MU_ERR_UNSUPPORTED, "attention_paged: dtype not implemented (float32, bfloat16)");
  if (B > MU_ATTENTION_PAGED_MAX_REQUESTS)
    return mu_set_error(ctx, MU_ERR_SIZE, "attention_paged: more than MU_ATTENTION_PAGED_MAX_REQUESTS requests");
  if (1ll * num_pages * page_size > INT_MAX || 1ll * n_tokens * Hq > INT_MAX)
    return mu_set_error(ctx, MU_ERR_SIZE, "attention_paged: slots or rows beyond 32 bits");
  if (q_ld < 1ll * Hq * D || out_ld < 1ll * Hq * D)
    return mu_set_error(ctx, MU_ERR_INVALID, "attention_paged: row stride below Hq * D");
  if (B == 0 || n_tokens == 0)
    return MU_OK;
  if (!q || !out || !query_start || !seq_lens || (table_stride > 0 && !block_table) ||
      (num_pages > 0 && (!k_cache || !v_cache || !k_scale || !v_scale)))
    return mu_set_error(ctx, MU_ERR_INVALID, "attention_paged: null pointer");
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u)
    return mu_set_error(ctx, MU_ERR_INVALID, "attention_paged: the caches must be 16-byte aligned");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
      workspace_bytes < mu_attention_paged_workspace_bytes(ctx, n_tokens, B, Hq, Hkv, D, dtype))
    return mu_set_error(ctx, MU_ERR_INVALID, "attention_paged: workspace missing, misaligned or too small "
                        "(mu_attention_paged_workspace_bytes)");
  if (mu_ctx_select_device(ctx) != MU_OK)
    return mu_set_error(ctx, MU_ERR_CUDA, "attention_paged: cannot select device");
  mu::PagedArgs a{};
  a.q = q, a.out = out, a.q_ld = q_ld, a.out_ld = out_ld;
  a.kc = static_cast<const uint8_t *>(k_cache), a.vc = static_cast<const uint8_t *>(v_cache);
  a.ks = k_scale, a.vs = v_scale, a.table = block_table, a.table_stride = table_stride;
  a.query_start = query_start, a.seq_lens = seq_lens, a.B = B, a.n_tokens = n_tokens;
  a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv, a.D = D, a.num_pages = num_pages, a.page_size = page_size;
  a.causal = causal != 0, a.status = mu_ctx_status_ptr(ctx);
  a.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(D)));
  if (mu::launch_attention_paged(a, workspace, dtype, mu_ctx_num_sms(ctx), static_cast<cudaStream_t>(stream)))
    return mu_set_error(ctx, MU_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
  return MU_OK;
}

} // extern "C"
