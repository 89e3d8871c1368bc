// Attention over a paged KV cache held in e4m3 with one scale per page and head (layout: kv_cache.cu).
//
//   out[t, hq, :] = sum_j softmax_j( q[t, hq, :] . K[j, hk, :] / sqrt(D) ) V[j, hk, :],  hk = hq / G
//
// Token i of a request with n new tokens and `len` tokens in the cache sits at position len - n + i;
// causal attention lets it see j <= that position. A row that sees nothing gives zeros.
//
// Work split: a request's rows (token, head of the group) are cut into row tiles, its keys into chunks;
// (request, KV head, row tile, chunk) in this order is one long list of units that the resident workers
// (warps of the tensor-core kernel, CTAs of the CUDA-core one) share out evenly, whatever the lengths
// are. A worker walks its range as segments, one per (request, head, row tile). A segment that covers
// all chunks writes its rows; one that does not leaves (running maximum, sum, weighted values) in the
// workspace, and a second small kernel joins the pieces. No atomics: results do not depend on the order
// in which workers run. (A causal row tile counts all of its request's chunks, those that it does not see among
// them. Prompts that take this file's kernels, float32 or head sizes other than 64 and 128, are therefore shared out
// unevenly: the workers of early rows have less to do.) Every item counts a few units more than its chunks,
// for what starting a segment costs: without it the workers that got many short requests finished last.
#include "../../include/munet_b200.h"
#include "attention_paged.cuh"
#include <climits>
#include <cmath>
#include <type_traits>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace mu {

template <int CHUNK> __device__ __forceinline__ int chunks_of(const Seq &s) {
  return s.seen > 0 ? (s.seen - 1) / CHUNK + 1 : 1;
}
template <int R, int CHUNK> __device__ __forceinline__ long long units_of(const PagedArgs &a, const Seq &s) {
  if (s.nq <= 0)
    return 0;
  const unsigned rows = static_cast<unsigned>(s.nq) * a.G; // n_tokens * Hq fits 31 bits
  return 1ll * a.Hkv * ((rows + R - 1) / R) * (chunks_of<CHUNK>(s) + START_UNITS);
}
// Inclusive prefix of units over the requests into shared memory; returns the total.
template <int THREADS, int R, int CHUNK>
__device__ __forceinline__ long long scan_units(const PagedArgs &a, long long *upto, long long *warp_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) {
    sum += units_of<R, CHUNK>(a, load_seq(a, b));
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

// Walks one worker's share of the unit list.
template <int R, int CHUNK> struct Walk {
  long long u, end, total;
  int workers, me, b;
  bool first;
  __device__ __forceinline__ Walk(long long total_, int me_, int workers_) : total(total_), me(me_), b(0), first(true) {
    workers = static_cast<int>(min(static_cast<long long>(workers_), total_)); // every active one has a unit
    u = end = 0;
    if (me < workers) { // start(w) = floor(total * w / workers)
      int rest;
      const long long each = div_rem(total, workers, rest);
      u = each * me + static_cast<unsigned>(rest * me) / static_cast<unsigned>(workers);
      end = each * (me + 1) + static_cast<unsigned>(rest * (me + 1)) / static_cast<unsigned>(workers);
    }
  }
  // the worker that holds unit x: the largest w with total * w < (x + 1) * workers
  __device__ __forceinline__ int owner(long long x) const {
    return static_cast<int>(div64((x + 1) * workers - 1, total));
  }
  // The next segment. `leader`: the thread that notes down a split item.
  __device__ __forceinline__ bool next(const PagedArgs &a, const long long *upto, Segment &g, Seq &s, bool leader) {
    int rows, tiles, nc, at, to;
    do { // more than once only where this worker's share ends inside an item's starting units
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
      rows = s.nq * a.G, tiles = (rows + R - 1) / R, nc = chunks_of<CHUNK>(s);
      const long long item = div_rem(u - (b ? upto[b - 1] : 0), nc + START_UNITS, at);
      int tile;
      g.head = static_cast<int>(div_rem(item, tiles, tile));
      g.row0 = tile * R;
      to = static_cast<int>(min(static_cast<long long>(nc + START_UNITS), at + (end - u)));
      u += to - at;
    } while (to <= START_UNITS);
    g.b = b;
    g.n_rows = min(rows - g.row0, R);
    g.chunk0 = max(at - START_UNITS, 0);
    g.chunks = to - START_UNITS - g.chunk0;
    g.slot = -1;
    if (g.chunks < nc) {
      g.slot = 2 * me + (first ? 0 : 1);
      const long long item0 = u - to; // of the item's units
      if (leader && g.chunk0 == 0) {
        SplitItem it;
        it.first_slot = g.slot, it.last = owner(item0 + nc + START_UNITS - 1);
        it.row0 = g.row0, it.n_rows = g.n_rows, it.q0 = s.q0, it.head = g.head;
        a.items[me] = it, a.notes[me].x = g.n_rows;
      } else if (leader) {
        a.notes[me].y = owner(item0 + START_UNITS);
      }
    }
    first = false;
    return true;
  }
};

// ---- CUDA-core kernel: head sizes that are no multiple of 16 ---------------------------------------
// float32 products and sums. Per warp a tile of 32 keys: for the scores a lane owns a key (its row is D
// consecutive bytes), for the weighted values a lane owns four dimensions (one, where D is odd).
// VB: bytes per load (4 or 1 by the head size), RT rows share every key, NA units per lane. Bound by the conversion
// and fp32 products: 32 requests of 2048 keys, 8 heads of 100, bfloat16: 80 us (105 MB: 1.3 TB/s); of 40: 33 us.
constexpr int SIMT_WARPS = 4, SIMT_THREADS = 32 * SIMT_WARPS, SIMT_CHUNK = 32 * SIMT_WARPS;

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
    a.notes[blockIdx.x] = make_int2(0, -1);
  const long long total = scan_units<SIMT_THREADS, RT, SIMT_CHUNK>(a, upto, warp_sum);
  if (total == 0)
    return;
  Walk<RT, SIMT_CHUNK> walk(total, blockIdx.x, gridDim.x);
  Segment g;
  Seq s;
  while (walk.next(a, upto, g, s, tid == 0)) {
    for (int e = tid; e < RT * Dq; e += SIMT_THREADS) {
      const int r = e / Dq, d = e - r * Dq;
      float v = 0.f;
      if (r < g.n_rows && d < a.D) {
        const int row = g.row0 + r;
        v = load_in(static_cast<const T *>(a.q) + (s.q0 + a.by_group.div(row)) * a.q_ld +
                    (1ll * g.head * a.G + a.by_group.mod(row)) * a.D + d);
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
      const int base = c * SIMT_CHUNK + warp * 32;
      if (base >= most)
        break;
      const int j = base + lane;
      long long row = -1;
      float kscale = 0.f, vscale = 0.f;
      if (j < most) {
        const int page = a.table[1ll * g.b * a.table_stride + a.by_page.div(j)];
        if (page >= 0 && page < a.num_pages) {
          const long long tile = 1ll * page * a.Hkv + g.head;
          row = tile * a.page_size + a.by_page.mod(j);
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
        if constexpr (VB == 4) {
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
        const int row = g.row0 + r;
        store_out(static_cast<T *>(a.out) + (s.q0 + a.by_group.div(row)) * a.out_ld +
                      (1ll * g.head * a.G + a.by_group.mod(row)) * a.D + d,
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

// ---- tensor-core kernel: head sizes that are multiples of 16 ----------------------------------------
// Bound by reading the cache (64 requests of up to 2048 keys, 16 heads of 128: 311 MB in 66 us with the join,
// 4.7 TB/s; 7 TB/s between the first tile and the first warp's end). A warp walks its keys in tiles (32 of them, 16
// for head sizes above 128), copies a tile's K and V bytes into its own two stages of shared memory (cp.async, 16
// bytes a lane), turns them into fp16 in registers and multiplies with mma.m16n8k16. Where requests x KV heads are
// many, a warp is a worker of its own and nothing ever synchronises the CTA (TEAM 1). Where they are few, every
// item is cut into many pieces whose join would cost as much as the rest (3 requests x 2 heads: 296 pieces
// each); there the four warps of a CTA are one worker, take every fourth tile and join in shared memory
// (TEAM 4).
//
// The keys are the M side of both products, so that eight rows fill the N side: S' = K q' is 16 keys x 8
// rows, O' = V' P' is 16 dimensions x 8 rows (with the rows as M, half to 15/16 of every product would be
// thrown away for single tokens). P leaves the first product's layout for the second's by movmatrix.
// Both products may permute what they sum over and O' its rows, so operands are read straight from the
// bytes: lane (g, c) = (lane / 4, lane % 4) reads, of keys g and g + 8, dimensions [c D/4, (c+1) D/4), and,
// of keys 2c, 2c+1, 2c+8, 2c+9, dimensions [g D/8, (g+1) D/8).
//
// Numbers: e4m3 is exact in fp16. A query row is scaled by a power of two to at most 2^15, which keeps a
// bfloat16 mantissa exact. A page's K scale multiplies its fp32 scores. Its V scale goes into the weight:
// with t = s + log2(vs), weights are 2^(t - max t + 15) in fp16 (so that a page of small values that
// matters keeps its bits above fp16's subnormals), and the softmax sum takes w / vs back out in fp32.
// SPLIT (float32): queries and weights are the sum of two fp16 numbers, 22 bits, and every product starts
// from zero and is added in fp32, because the tensor core rounds its running sum towards zero.
constexpr float W_EXP = 15.f; // the largest weight of a row is 2^15: fp16 ends at 65504

template <int DP, int NR, int TEAM, bool SPLIT> struct MmaCfg {
  static constexpr int WARPS = 4, THREADS = 32 * WARPS;
  static constexpr int CTAS_PER_SM = (DP <= 128 && NR == 1) ? 3 : 2; // 12 or 8 warps: by their registers
  static constexpr int R = 8 * NR;
  static constexpr int TILE = DP <= 128 ? 32 : 16, CHUNK = TEAM * TILE, MT = TILE / 16;
  // bytes between keys: whole bank cycles are swizzled, others padded
  static constexpr int PITCH = DP == 64 || DP == 128 || DP == 256 ? DP : DP + 16;
  static constexpr int TILE_BYTES = TILE * PITCH, WARP_BYTES = 4 * TILE_BYTES; // K and V, two stages
  static_assert(TEAM == 1 || (TEAM == WARPS && WARP_BYTES >= R * DP * 4), "a warp's ring carries its rows to the join");
  static constexpr int KW = DP / 16, VW = DP / 32, NT = DP / 16; // 32-bit words of K / V a lane reads per key; d-tiles
};

// what is left of two floats after their rounding to fp16
__device__ __forceinline__ uint32_t f16x2_rest(float lo, float hi, uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  return f16x2(lo - f.x, hi - f.y);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
// 16 bytes into shared memory, or 16 zero bytes
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// byte offset of 16-byte chunk `chunk` of key `row` in a tile
template <int DP, int PITCH> __device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
  if constexpr (DP == 128 || DP == 256)
    return row * PITCH + ((chunk ^ (row & 7)) << 4);
  else if constexpr (DP == 64)
    return row * PITCH + ((chunk ^ ((row >> 1) & 3)) << 4);
  else
    return row * PITCH + (chunk << 4);
}
// N 32-bit words from byte `byte` (a multiple of 4 N, of 4 or of 8) of key `row`
template <int DP, int PITCH, int N>
__device__ __forceinline__ void read_words(uint32_t (&w)[N], const unsigned char *tile, int row, int byte) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 u = *reinterpret_cast<const uint4 *>(tile + tile_at<DP, PITCH>(row, byte / 16 + i));
      w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const int at = byte + 8 * i;
      const uint2 u = *reinterpret_cast<const uint2 *>(tile + tile_at<DP, PITCH>(row, at / 16) + at % 16);
      w[2 * i] = u.x, w[2 * i + 1] = u.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = byte + 4 * i;
      w[i] = *reinterpret_cast<const uint32_t *>(tile + tile_at<DP, PITCH>(row, at / 16) + at % 16);
    }
  }
}
template <typename T, int DP, int NR, int TEAM>
__global__ void __launch_bounds__(MmaCfg<DP, NR, TEAM, sizeof(T) == 4>::THREADS,
                                  MmaCfg<DP, NR, TEAM, sizeof(T) == 4>::CTAS_PER_SM)
    attention_paged_mma_kernel(PagedArgs a) {
  constexpr bool SPLIT = sizeof(T) == 4;
  using Cfg = MmaCfg<DP, NR, TEAM, SPLIT>;
  constexpr int KW = Cfg::KW, VW = Cfg::VW, NT = Cfg::NT, MT = Cfg::MT, TILE = Cfg::TILE, R = Cfg::R;
  constexpr int PITCH = Cfg::PITCH, NS = SPLIT ? 2 : 1;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ long long warp_sum[Cfg::WARPS];
  __shared__ float2 team_ml[TEAM][R];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = lane >> 2, quad = lane & 3;
  unsigned char *ring = smem_raw + warp * Cfg::WARP_BYTES;
  long long *upto = reinterpret_cast<long long *>(smem_raw + Cfg::WARPS * Cfg::WARP_BYTES);
  const uint32_t ring_u32 = smem_u32(ring);

  // neighbouring workers sit on different SMs, so that a short list spreads out
  const int me = TEAM == 1 ? warp * gridDim.x + blockIdx.x : blockIdx.x;
  const bool leader = TEAM == 1 ? lane == 0 : tid == 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // the join waits for the whole grid anyway
  if (leader)
    a.notes[me] = make_int2(0, -1);
  __syncwarp();
  const long long total = scan_units<Cfg::THREADS, R, Cfg::CHUNK>(a, upto, warp_sum);
  if (total == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory"); // see the end
    return;
  }
  Walk<R, Cfg::CHUNK> walk(total, me, gridDim.x * (Cfg::WARPS / TEAM));
  const int D = a.D;
  // The walk as a stream of batches: up to 32 half tiles of one segment, whose pages and scales the lanes
  // hold. The batch after the current one is looked up while that runs, in steps that do not wait for one
  // another's loads (table, then scales), and its first tile is on its way before the current one is done:
  // a segment begun cold cost 5.6 us of dependent loads.
  constexpr int BATCH = 32 / MT, STEP = TEAM * TILE; // tiles of a batch; keys between a warp's tiles
  struct Batch {
    int head, row0, n_rows, slot, q0, nq, len, seen;
    int key0, tiles;
    int page;     // of half tile `lane`; -1: none
    float ks, vs; // its scales; vs 0: no page
    bool first, last;
  };
  Segment g;
  Seq s;
  int seg_key = 0, seg_end = 0; // this warp's keys of segment (g, s) that have not been handed out
  bool open = false;            // some batch of it is still to come
  auto half_key = [&](const Batch &n) { return n.key0 + (lane / MT) * STEP + (lane % MT) * 16; };
  auto fetch = [&](Batch &n) -> bool {
    n.first = !open;
    if (!open) {
      if (!walk.next(a, upto, g, s, leader))
        return false;
      seg_key = g.chunk0 * Cfg::CHUNK + (TEAM == 1 ? 0 : warp * TILE);
      seg_end = min(row_limit(a, s, g.row0 + g.n_rows - 1), (g.chunk0 + g.chunks) * Cfg::CHUNK);
      const int r = g.row0 + grp; // its queries: into L1
      if (grp < g.n_rows)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const T *>(a.q) + (s.q0 + a.by_group.div(r)) * a.q_ld +
                                                    (1ll * g.head * a.G + a.by_group.mod(r)) * D + quad * D / 4));
    }
    n.head = g.head, n.row0 = g.row0, n.n_rows = g.n_rows, n.slot = g.slot;
    n.q0 = s.q0, n.nq = s.nq, n.len = s.len, n.seen = s.seen;
    n.key0 = seg_key;
    n.tiles = seg_end > seg_key ? min(BATCH, (seg_end - seg_key + STEP - 1) / STEP) : 0;
    const int key = half_key(n);
    n.page = -2; // not looked for
    if (lane / MT < n.tiles && key < seg_end)
      n.page = a.table[1ll * g.b * a.table_stride + a.by_page.div(key)];
    seg_key += BATCH * STEP;
    open = seg_key < seg_end;
    n.last = !open;
    return true;
  };
  auto scales = [&](Batch &n) { // the pages have arrived
    n.ks = n.vs = 0.f;
    if (n.page >= 0 && n.page < a.num_pages) {
      const long long t = 1ll * n.page * a.Hkv + n.head;
      n.ks = a.ks[t], n.vs = a.vs[t];
    } else {
      if (n.page != -2)
        atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
      n.page = -1;
    }
  };
  auto issue = [&](const Batch &n, int i, int stage) {
    if (i < n.tiles) {
      const uint32_t st = ring_u32 + stage * 2 * Cfg::TILE_BYTES;
#pragma unroll
      for (int hf = 0; hf < MT; ++hf) {
        const int page = __shfl_sync(~0u, n.page, i * MT + hf);
        const int key = n.key0 + i * STEP + 16 * hf, live = page >= 0 ? n.seen - key : 0; // behind it: anything
        const int in_page = a.by_page.mod(key);
        const long long off = page >= 0 ? ((1ll * page * a.Hkv + n.head) * a.page_size + in_page) * D : 0;
        if (D == DP && live >= 16) { // sixteen whole rows: one run of bytes
          const uint8_t *kp = a.kc + off + lane * 16, *vp = a.vc + off + lane * 16;
#pragma unroll
          for (int j = 0; j < DP / 32; ++j) {
            const int idx = lane + 32 * j;
            const uint32_t at = st + tile_at<DP, PITCH>(hf * 16 + idx / (DP / 16), idx % (DP / 16));
            cp_async16(at, kp + 512 * j);
            cp_async16(at + Cfg::TILE_BYTES, vp + 512 * j);
          }
        } else {
#pragma unroll
          for (int j = 0; j < DP / 32; ++j) {
            const int idx = lane + 32 * j, row = idx / (DP / 16), chunk = idx % (DP / 16);
            const uint32_t at = st + tile_at<DP, PITCH>(hf * 16 + row, chunk);
            const bool real = row < live && chunk * 16 < D;
            const long long o = real ? off + row * D + chunk * 16 : 0;
            cp_async16(at, a.kc + o, real);
            cp_async16(at + Cfg::TILE_BYTES, a.vc + o, real);
          }
        }
      }
    }
    cp_async_commit();
  };

  uint32_t qf[NS][NR][KW][2]; // queries: fp16 fragments, and each row's factor back
  float fac[NR][2];
  float o[NR][NT][4], m[NR][2], l[NR][2];
  int lim[NR][2], least = 0; // keys that this lane's rows (rb * 8 + 2 quad + e) see, and the least over all rows
  int stage = 0;
  Batch cur, nxt;
  bool more = fetch(cur);
  if (more) {
    scales(cur);
    issue(cur, 0, stage);
  }
  bool ahead = true; // the first tile of `cur` is on its way, its scales are too
  while (more) {
    const bool more_after = fetch(nxt);
    if (!more_after)
      nxt.tiles = 0, nxt.page = -2;
    if (!ahead) {
      scales(cur);
      issue(cur, 0, stage);
    }
    if (cur.first) {
      const Seq cs{cur.q0, cur.nq, cur.len, cur.seen};
      least = row_limit(a, cs, cur.row0);
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        m[rb][0] = m[rb][1] = -INFINITY, l[rb][0] = l[rb][1] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          lim[rb][e] = row_limit(a, cs, cur.row0 + rb * 8 + quad * 2 + e);
#pragma unroll
        for (int j = 0; j < NT; ++j)
          o[rb][j][0] = o[rb][j][1] = o[rb][j][2] = o[rb][j][3] = 0.f;
      }
      float qv[NR][DP / 4];
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        const int r = rb * 8 + grp, row = cur.row0 + r;
        const bool live = r < cur.n_rows;
        const T *qp = static_cast<const T *>(a.q) +
                      (live ? (cur.q0 + a.by_group.div(row)) * a.q_ld + (1ll * cur.head * a.G + a.by_group.mod(row)) * D : 0);
        const bool vec = (reinterpret_cast<uintptr_t>(qp) & 7u) == 0;
        float (&v)[DP / 4] = qv[rb];
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          const int d = quad * (DP / 4) + 4 * i;
          if (live && d < D) {
            if (vec && sizeof(T) == 2) {
              const uint2 u = *reinterpret_cast<const uint2 *>(qp + d);
              v[4 * i] = bf16_lo(u.x), v[4 * i + 1] = bf16_hi(u.x), v[4 * i + 2] = bf16_lo(u.y), v[4 * i + 3] = bf16_hi(u.y);
            } else if (vec) {
              const float2 x = *reinterpret_cast<const float2 *>(qp + d), y = *reinterpret_cast<const float2 *>(qp + d + 2);
              v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = y.x, v[4 * i + 3] = y.y;
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                v[4 * i + j] = load_in(qp + d + j);
            }
          } else {
            v[4 * i] = v[4 * i + 1] = v[4 * i + 2] = v[4 * i + 3] = 0.f;
          }
        }
      }

#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        const float (&v)[DP / 4] = qv[rb];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < DP / 4; ++i)
          top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(~0u, top, 1));
        top = max(top, __shfl_xor_sync(~0u, top, 2));
        const int e = min(max(static_cast<int>(top >> 23) - 127 - 14, -100), 113);
        const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        const float back = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        fac[rb][0] = __shfl_sync(~0u, back, quad * 8) * a.scale_log2; // row 2 quad: lanes 8 quad ..
        fac[rb][1] = __shfl_sync(~0u, back, quad * 8 + 4) * a.scale_log2;
#pragma unroll
        for (int i = 0; i < KW; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = v[4 * i + 2 * h] * f, y = v[4 * i + 2 * h + 1] * f;
            qf[0][rb][i][h] = f16x2(x, y);
            if constexpr (SPLIT)
              qf[NS - 1][rb][i][h] = f16x2_rest(x, y, qf[0][rb][i][h]);
          }
      }
    }

    // log2 and reciprocal of the V scales; no page: no weight
    const float my_vs = fmaxf(cur.vs, 0x1p-64f);
    const float my_lv = cur.page >= 0 ? log2f(my_vs) : -INFINITY, my_iv = cur.page >= 0 ? 1.f / my_vs : 0.f;

    ahead = false;
    for (int i = 0; i < cur.tiles; ++i) {
      if (i + 1 < cur.tiles) {
        issue(cur, i + 1, stage ^ 1);
      } else if (TEAM == 1 || !cur.last) {
        scales(nxt);
        issue(nxt, 0, stage ^ 1);
        ahead = true;
      } else {
        cp_async_commit(); // the ring is needed for the join
      }
      cp_async_wait<1>();
      __syncwarp();
      const unsigned char *kt = ring + stage * 2 * Cfg::TILE_BYTES, *vt = kt + Cfg::TILE_BYTES;
      const int key0 = cur.key0 + i * STEP;
      const bool edge = key0 + TILE > least;

      // scores, in units of log2, with log2 of the V scale
      float sc[NR][MT][4], iv[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t w0[KW], w1[KW];
        read_words<DP, PITCH, KW>(w0, kt, mt * 16 + grp, quad * (DP / 4));
        read_words<DP, PITCH, KW>(w1, kt, mt * 16 + grp + 8, quad * (DP / 4));
#pragma unroll
        for (int rb = 0; rb < NR; ++rb)
          sc[rb][mt][0] = sc[rb][mt][1] = sc[rb][mt][2] = sc[rb][mt][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          const uint32_t ka[4] = {f16x2_of_e4m3_lo(w0[k]), f16x2_of_e4m3_lo(w1[k]), f16x2_of_e4m3_hi(w0[k]),
                                  f16x2_of_e4m3_hi(w1[k])};
#pragma unroll
          for (int rb = 0; rb < NR; ++rb) {
            if constexpr (SPLIT) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(c, ka, qf[NS - 1][rb][k][0], qf[NS - 1][rb][k][1]);
              mma_f16(c, ka, qf[0][rb][k][0], qf[0][rb][k][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sc[rb][mt][e] += c[e];
            } else {
              mma_f16(sc[rb][mt], ka, qf[0][rb][k][0], qf[0][rb][k][1]);
            }
          }
        }
        const int src = i * MT + mt;
        const float ks = __shfl_sync(~0u, cur.ks, src), lv = __shfl_sync(~0u, my_lv, src);
        iv[mt] = __shfl_sync(~0u, my_iv, src);
#pragma unroll
        for (int rb = 0; rb < NR; ++rb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[rb][mt][e] = fmaf(sc[rb][mt][e], ks * fac[rb][e & 1], lv);
            if (edge && key0 + mt * 16 + grp + 8 * (e >> 1) >= lim[rb][e & 1])
              sc[rb][mt][e] = -INFINITY;
          }
      }

      uint32_t pf[NS][NR][MT][2];
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        float t[2], ref[2];
        bool grew = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          t[e] = m[rb][e];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            t[e] = fmaxf(t[e], fmaxf(sc[rb][mt][e], sc[rb][mt][e + 2]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1)
            t[e] = fmaxf(t[e], __shfl_xor_sync(~0u, t[e], d));
          ref[e] = t[e] == -INFINITY ? 0.f : t[e] - W_EXP;
          grew |= t[e] != m[rb][e];
        }
        if (__any_sync(~0u, grew)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = m[rb][e] == -INFINITY ? 0.f : ex2_approx(m[rb][e] - t[e]);
            l[rb][e] *= f, m[rb][e] = t[e];
#pragma unroll
            for (int j = 0; j < NT; ++j)
              o[rb][j][e] *= f, o[rb][j][e + 2] *= f;
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float (&x)[4] = sc[rb][mt];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = ex2_approx(x[e] - ref[e & 1]);
          l[rb][0] = fmaf(x[0] + x[2], iv[mt], l[rb][0]), l[rb][1] = fmaf(x[1] + x[3], iv[mt], l[rb][1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t hi = f16x2(x[2 * h], x[2 * h + 1]);
            pf[0][rb][mt][h] = transpose8x8(hi);
            if constexpr (SPLIT)
              pf[NS - 1][rb][mt][h] = transpose8x8(f16x2_rest(x[2 * h], x[2 * h + 1], hi));
          }
        }
      }

#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t w[4][VW]; // keys 2 quad, 2 quad + 1, and both + 8
#pragma unroll
        for (int r = 0; r < 4; ++r)
          read_words<DP, PITCH, VW>(w[r], vt, mt * 16 + 2 * quad + (r & 1) + 8 * (r >> 1), grp * (DP / 8));
        // dimensions 2j and 2j + 1 of this lane's for two keys side by side
        auto values = [&](const uint32_t (&x)[4][VW], int j, uint32_t (&va)[4]) {
          const uint32_t sel = j & 1 ? 0x7362 : 0x5140;
          const uint32_t b0 = __byte_perm(x[0][j >> 1], x[1][j >> 1], sel), b1 = __byte_perm(x[2][j >> 1], x[3][j >> 1], sel);
          va[0] = f16x2_of_e4m3_lo(b0), va[1] = f16x2_of_e4m3_hi(b0);
          va[2] = f16x2_of_e4m3_lo(b1), va[3] = f16x2_of_e4m3_hi(b1);
        };
        bool nan = false;
        if (edge) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int q = 0; q < VW; ++q)
              nan |= has_nan_e4m3(w[r][q]);
          nan = __any_sync(~0u, nan);
        }
        if (!nan) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            uint32_t va[4];
            values(w, j, va);
#pragma unroll
            for (int rb = 0; rb < NR; ++rb) {
              if constexpr (SPLIT) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(c, va, pf[NS - 1][rb][mt][0], pf[NS - 1][rb][mt][1]);
                mma_f16(c, va, pf[0][rb][mt][0], pf[0][rb][mt][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  o[rb][j][e] += c[e];
              } else {
                mma_f16(o[rb][j], va, pf[0][rb][mt][0], pf[0][rb][mt][1]);
              }
            }
          }
        } else {
          // A NaN among keys that some rows may not see: zero weights would not keep it out, so the keys go
          // one at a time and a row takes only those it sees.
#pragma unroll 1
          for (int t = 0; t < 16; ++t) {
            const int key = key0 + mt * 16 + t;
            uint32_t x[4][VW];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int q = 0; q < VW; ++q)
                x[r][q] = t == 2 * quad + (r & 1) + 8 * (r >> 1) ? w[r][q] : 0u;
            const uint32_t keep = (t & 7) >> 1 == quad ? (t & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
            const uint32_t k0 = t < 8 ? keep : 0u, k1 = t < 8 ? 0u : keep;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              uint32_t va[4];
              values(x, j, va);
#pragma unroll
              for (int rb = 0; rb < NR; ++rb) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = NS - 1; n >= 0; --n)
                  mma_f16(c, va, pf[n][rb][mt][0] & k0, pf[n][rb][mt][1] & k1);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (key < lim[rb][e & 1])
                    o[rb][j][e] += c[e];
              }
            }
          }
        }
      }
      __syncwarp(); // the stage may be overwritten
      stage ^= 1;
    }

    if constexpr (TEAM > 1) {
      if (cur.last) { // every warp's rows through its ring, then the CTA joins them
        cp_async_wait<0>();
        __syncwarp();
        float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
        for (int rb = 0; rb < NR; ++rb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float sum = l[rb][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
              sum += __shfl_xor_sync(~0u, sum, d);
            const int r = rb * 8 + quad * 2 + e;
            if (grp == 0)
              team_ml[warp][r] = make_float2(m[rb][e] - W_EXP, sum);
            if (r < cur.n_rows)
#pragma unroll
              for (int j = 0; j < NT; ++j)
                *reinterpret_cast<float2 *>(mine + r * DP + grp * (DP / 8) + 2 * j) = make_float2(o[rb][j][e], o[rb][j][e + 2]);
          }
        __syncthreads();
        for (int r = warp; r < cur.n_rows; r += Cfg::WARPS) {
          float M = -INFINITY, sum = 0.f, w[Cfg::WARPS];
#pragma unroll
          for (int t = 0; t < Cfg::WARPS; ++t)
            M = fmaxf(M, team_ml[t][r].x);
#pragma unroll
          for (int t = 0; t < Cfg::WARPS; ++t) {
            w[t] = rel_weight(team_ml[t][r].x, M);
            sum = fmaf(w[t], team_ml[t][r].y, sum);
          }
          const int row = cur.row0 + r;
          const long long pr = 1ll * cur.slot * R + r;
          T *p = static_cast<T *>(a.out) + (cur.q0 + a.by_group.div(row)) * a.out_ld + (1ll * cur.head * a.G + a.by_group.mod(row)) * D;
          for (int d = lane; d < D; d += 32) {
            float x = 0.f;
#pragma unroll
            for (int t = 0; t < Cfg::WARPS; ++t)
              x = fmaf(w[t], reinterpret_cast<const float *>(smem_raw + t * Cfg::WARP_BYTES)[r * DP + d], x);
            if (cur.slot < 0)
              store_out(p + d, sum == 0.f ? 0.f : x / sum);
            else
              a.part_o[pr * D + d] = x;
          }
          if (cur.slot >= 0 && lane == 0)
            a.part_ml[pr] = make_float2(M, sum);
        }
        __syncthreads(); // the rings are free again
      }
    } else if (cur.last) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[rb][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1)
            sum += __shfl_xor_sync(~0u, sum, d);
          const int r = rb * 8 + quad * 2 + e;
          if (r >= cur.n_rows)
            continue;
          if (cur.slot < 0) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int row = cur.row0 + r;
            T *p = static_cast<T *>(a.out) + (cur.q0 + a.by_group.div(row)) * a.out_ld + (1ll * cur.head * a.G + a.by_group.mod(row)) * D;
            const bool vec = (reinterpret_cast<uintptr_t>(p) & (2 * sizeof(T) - 1)) == 0;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const int d = grp * (DP / 8) + 2 * j;
              // the reciprocal is off by half a unit; float32 takes the quotient
              const float x = SPLIT ? (sum == 0.f ? 0.f : o[rb][j][e] / sum) : o[rb][j][e] * inv;
              const float y = SPLIT ? (sum == 0.f ? 0.f : o[rb][j][e + 2] / sum) : o[rb][j][e + 2] * inv;
              if (d >= D)
                continue;
              if (vec && sizeof(T) == 2) {
                *reinterpret_cast<uint32_t *>(p + d) = pack_bf16x2(x, y);
              } else if (vec) {
                *reinterpret_cast<float2 *>(p + d) = make_float2(x, y);
              } else {
                store_out(p + d, x), store_out(p + d + 1, y);
              }
            }
          } else {
            const long long pr = 1ll * cur.slot * R + r;
            if (grp == 0)
              a.part_ml[pr] = make_float2(m[rb][e] - W_EXP, sum);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const int d = grp * (DP / 8) + 2 * j;
              if (d < D)
                *reinterpret_cast<float2 *>(a.part_o + pr * D + d) = make_float2(o[rb][j][e], o[rb][j][e + 2]);
            }
          }
        }
      __syncwarp();
    }
    cur = nxt, more = more_after;
  }
  cp_async_wait<0>();
  // Behind the prompt-chunk kernel this one starts while that drains and reads nothing of it; the join, which waits for
  // this grid, needs both.
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- joining the pieces ---------------------------------------------------------------------------
// The rows of an item with P pieces are dealt out to the first P workers that have a piece of it, so that
// one long request is not joined in one place; a CTA stands for one worker of the main kernel or for four.
// Time here is latency (note -> item -> maxima -> rows; 3 to 4 us behind a decode step of 64 requests), so every
// step loads all it needs at once. Launched so that it may become resident while the main kernel drains;
// griddepcontrol.wait orders its reads after that kernel's writes (loads go to L2: a line of an earlier call's pieces
// may still be in L1).
constexpr int JOIN_THREADS = 128, JOIN_WARPS = JOIN_THREADS / 32, JOIN_DIMS = 8; // dimensions per lane: D <= 256

// Where lane `lane` keeps dimension v of its JOIN_DIMS: four in a row where rows are whole 16-byte words.
__device__ __forceinline__ int join_dim(int D, int lane, int v) {
  return D % 4 == 0 ? (v >> 2) * 128 + lane * 4 + (v & 3) : lane + 32 * v;
}
struct Joined {
  float M, sum, o[JOIN_DIMS];
};
// Pieces first, first + step, ... of one row, by one warp.
__device__ __forceinline__ Joined join_pieces(const PagedArgs &a, const SplitItem &it, int owner, int r, int first, int step,
                                              int pieces) {
  const int lane = threadIdx.x & 31;
  Joined j;
  j.M = -INFINITY, j.sum = 0.f;
#pragma unroll
  for (int v = 0; v < JOIN_DIMS; ++v)
    j.o[v] = 0.f;
  auto row_of = [&](int i) { return 1ll * (i == 0 ? it.first_slot : 2 * (owner + i)) * a.rows_per_tile + r; };
  for (int p0 = first; p0 < pieces; p0 += 32 * step) {
    const int mine = p0 + lane * step;
    const float2 ml = mine < pieces ? __ldcg(a.part_ml + row_of(mine)) : make_float2(-INFINITY, 0.f);
    float top = fmaxf(ml.x, j.M);
#pragma unroll
    for (int d = 16; d; d >>= 1)
      top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const float old = rel_weight(j.M, top), h = mine < pieces ? rel_weight(ml.x, top) : 0.f;
    float sum = mine < pieces ? h * ml.y : 0.f;
#pragma unroll
    for (int d = 16; d; d >>= 1)
      sum += __shfl_xor_sync(~0u, sum, d);
    j.sum = j.sum * old + sum, j.M = top;
#pragma unroll
    for (int v = 0; v < JOIN_DIMS; ++v)
      j.o[v] *= old;
    const int n = min(32, (pieces - p0 + step - 1) / step);
    auto add = [&](auto dims, auto count, int i0) { // some pieces, their loads first
      constexpr int V = decltype(dims)::value, E = decltype(count)::value;
      float x[E][V];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float *src = a.part_o + row_of(p0 + min(i0 + e, n - 1) * step) * a.D;
        if (a.D % 4 == 0) {
#pragma unroll
          for (int v = 0; v < V; v += 4) {
            const int d = join_dim(a.D, lane, v);
            const float4 q = d < a.D ? __ldcg(reinterpret_cast<const float4 *>(src + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[e][v] = q.x, x[e][v + 1] = q.y, x[e][v + 2] = q.z, x[e][v + 3] = q.w;
          }
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v)
            x[e][v] = lane + 32 * v < a.D ? __ldcg(src + lane + 32 * v) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float w = __shfl_sync(~0u, h, min(i0 + e, 31));
        if (i0 + e < n)
#pragma unroll
          for (int v = 0; v < V; ++v)
            j.o[v] = fmaf(w, x[e][v], j.o[v]);
      }
    };
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, JOIN_DIMS>;
    if (a.D > 128) {
      for (int i0 = 0; i0 < n; i0 += 8)
        add(Eight{}, Eight{}, i0);
    } else if (n <= 4) {
      add(Four{}, Four{}, 0);
    } else {
      for (int i0 = 0; i0 < n; i0 += 16)
        add(Four{}, std::integral_constant<int, 16>{}, i0);
    }
  }
  return j;
}

// The workers of one main kernel: a CTA of the join stands for `per_cta` of them (1 or JOIN_WARPS), `ctas` CTAs share
// the rows of one.
struct JoinShare {
  int workers, per_cta, ctas; // one of the last two is 1
  int blocks() const { return (workers + per_cta - 1) / per_cta * ctas; }
};
// CTA (bx, by) of the join
template <typename T>
__device__ __forceinline__ void join_rows(const PagedArgs &a, int workers, int per_cta, int ctas, int bx, int by) {
  __shared__ float red_o[JOIN_WARPS][32 * JOIN_DIMS];
  __shared__ float2 red_ml[JOIN_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto note_of = [&](int w) { return __ldcg(a.notes + w); };
  auto item_of = [&](int w) {
    const int2 *p = reinterpret_cast<const int2 *>(a.items + w);
    const int2 x = __ldcg(p), y = __ldcg(p + 1), z = __ldcg(p + 2);
    return SplitItem{x.x, x.y, y.x, y.y, z.x, z.y};
  };
  static_assert(sizeof(SplitItem) == 24, "three pairs");
  auto out_row = [&](const SplitItem &it, int r) {
    const int row = it.row0 + r;
    return static_cast<T *>(a.out) + (it.q0 + a.by_group.div(row)) * a.out_ld + (1ll * it.head * a.G + a.by_group.mod(row)) * a.D;
  };
  constexpr int FEW = 16;
  // Few pieces: a warp joins a row. With one worker to the CTA its warps share the rows, with four each has
  // a worker of its own.
  {
    const int me = bx * per_cta + (per_cta > 1 ? warp : 0);
    const int part = per_cta > 1 ? 0 : by * JOIN_WARPS + warp, parts = per_cta > 1 ? 1 : ctas * JOIN_WARPS;
    const int2 note = me < workers ? note_of(me) : make_int2(0, -1);
    bool many = false;
#pragma unroll 1
    for (int job = 0; job < 2; ++job) { // the item this worker began, the one its first segment continued
      const int owner = job == 0 ? me : note.y;
      if (job == 0 ? note.x == 0 : note.y < 0)
        continue;
      const SplitItem it = item_of(owner);
      const int pieces = it.last - owner + 1, share = min(pieces, it.n_rows);
      if (pieces > FEW) {
        many = true;
        continue;
      }
      for (int r = me - owner + part * share; r < it.n_rows; r += parts * share) {
        const Joined j = join_pieces(a, it, owner, r, 0, 1, pieces);
        T *out = out_row(it, r);
#pragma unroll
        for (int v = 0; v < JOIN_DIMS; ++v)
          if (const int d = join_dim(a.D, lane, v); d < a.D)
            store_out(out + d, j.sum == 0.f ? 0.f : j.o[v] / j.sum);
      }
    }
    if (!__syncthreads_or(many))
      return;
  }
  // Many pieces: all warps join a row.
#pragma unroll 1
  for (int me = bx * per_cta; me < min((bx + 1) * per_cta, workers); ++me) {
    const int2 note = note_of(me);
#pragma unroll 1
    for (int job = 0; job < 2; ++job) {
      const int owner = job == 0 ? me : note.y;
      if (job == 0 ? note.x == 0 : note.y < 0)
        continue;
      const SplitItem it = item_of(owner);
      const int pieces = it.last - owner + 1, share = min(pieces, it.n_rows);
      if (pieces <= FEW)
        continue;
      for (int r = me - owner + by * share; r < it.n_rows; r += ctas * share) {
        const Joined j = join_pieces(a, it, owner, r, warp, JOIN_WARPS, pieces);
        if (lane == 0)
          red_ml[warp] = make_float2(j.M, j.sum);
#pragma unroll
        for (int v = 0; v < JOIN_DIMS; ++v)
          red_o[warp][join_dim(a.D, lane, v)] = j.o[v];
        __syncthreads();
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w)
          M = fmaxf(M, red_ml[w].x);
        for (int d = tid; d < a.D; d += JOIN_THREADS) {
          float all = 0.f, x = 0.f;
#pragma unroll
          for (int w = 0; w < JOIN_WARPS; ++w) {
            const float f = rel_weight(red_ml[w].x, M);
            all += f * red_ml[w].y, x += f * red_o[w][d];
          }
          store_out(out_row(it, r) + d, all == 0.f ? 0.f : x / all);
        }
        __syncthreads();
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) attention_paged_join_kernel(PagedArgs a, JoinShare n) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  join_rows<T>(a, n.workers, n.per_cta, 1, blockIdx.x, 0);
}
// Both main kernels' pieces: two joins one after the other would be twice the latency.
template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS)
    attention_paged_join_both_kernel(PagedArgs a, JoinShare n, int blocks, PagedArgs b, JoinShare m) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int block = blockIdx.x;
  if (block < blocks)
    join_rows<T>(a, n.workers, 1, n.ctas, block / n.ctas, block % n.ctas);
  else
    join_rows<T>(b, m.workers, m.per_cta, 1, block - blocks, 0);
}

// ---- host -----------------------------------------------------------------------------------------
constexpr int SIMT_CTAS_PER_SM = 4;
constexpr int MAX_WORKERS_PER_SM = 12;

// Rows of partial results per SM, two pieces a worker: 12 workers of 8 rows, 8 of 16, 4 CTAs of 8; one of 256
// for prompt chunks.
constexpr int MAX_PART_ROWS_PER_SM = 2 * 128;
// Requests with this many rows (new tokens x heads of a group) or more go to the prompt-chunk kernel: below, a
// tile of 256 rows would be mostly empty, and reading the keys once per 16 rows costs less (8 requests of 4096
// keys, 4 KV heads of 128: 64 rows 46 us against 50, 72 rows 51 against 51, 80 rows 60 against 51, 128 rows 83
// against 53; of 64: 72 rows 41 against 44, 80 rows 43 against 44, 88 rows 49 against 45: there the border lies 8 to 15
// rows higher, and one number serves both at a cost of 1 to 3 us). The host cannot see lengths: a call of more tokens than
// requests launches the prompt-chunk kernel whether or not a request has this many.
constexpr int TILE_KERNEL_ROWS = 73;
bool tile_kernel_shape(int n_tokens, int G, int D, int dtype) {
  return dtype == BF16 && (D == 64 || D == 128) && 1ll * n_tokens * G >= TILE_KERNEL_ROWS;
}
bool uses_tile_kernel(int n_tokens, int B, int G, int D, int dtype) {
  return tile_kernel_shape(n_tokens, G, D, dtype) && n_tokens > B && B <= MU_PAGED_TILE_MAX_REQUESTS;
}
// One kernel's part of the workspace: pieces, notes, split items.
size_t part_bytes(size_t rows, int D, int workers) {
  return (rows * (sizeof(float) * D + sizeof(float2)) + (sizeof(SplitItem) + sizeof(int2)) * workers + 63) & ~size_t(63);
}
size_t tile_part_bytes(int num_sms, int D) { return part_bytes(2ull * PAGED_TILE_ROWS * num_sms, D, num_sms); }
// Whatever the number of requests: a workspace for a program's largest call serves its smaller ones, among them those of
// few requests that use the prompt-chunk kernel where the largest does not.
size_t paged_workspace_bytes(int num_sms, int n_tokens, int G, int D, int dtype) {
  return part_bytes(1ull * MAX_PART_ROWS_PER_SM * num_sms, D, num_sms * MAX_WORKERS_PER_SM) +
         (n_tokens > 1 && tile_kernel_shape(n_tokens, G, D, dtype) ? tile_part_bytes(num_sms, D) : 0) + 64;
}
void place_parts(PagedArgs &a, unsigned char *w, size_t rows, int workers) {
  a.part_o = reinterpret_cast<float *>(w);
  w += sizeof(float) * rows * a.D;
  a.part_ml = reinterpret_cast<float2 *>(w);
  w += sizeof(float2) * rows;
  a.notes = reinterpret_cast<int2 *>(w);
  w += sizeof(int2) * workers;
  a.items = reinterpret_cast<SplitItem *>(w);
}

// A launch that may begin while the kernel before it in the stream drains.
template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), int grid, int threads, size_t smem, bool early, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at, cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? 0 : 2;
}
// `chunks`: the prompt-chunk kernel's arguments, where it went first
constexpr int TILE_JOIN_CTAS = 8;
template <typename T>
int launch_join(const PagedArgs &a, const JoinShare &n, const PagedArgs *chunks, int num_sms, cudaStream_t st) {
  if (!chunks)
    return launch_behind(attention_paged_join_kernel<T>, n.blocks(), JOIN_THREADS, 0, true, st, a, n);
  const JoinShare m{num_sms, 1, TILE_JOIN_CTAS};
  return launch_behind(attention_paged_join_both_kernel<T>, m.blocks() + n.blocks(), JOIN_THREADS, 0, true, st, *chunks, m,
                       m.blocks(), a, n);
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
  return launch_join<T>(a, JoinShare{ctas, 1, 1}, nullptr, num_sms, st);
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

template <typename T, int DP, int NR, int TEAM> int launch_mma_team(PagedArgs a, const PagedArgs *chunks, int num_sms, cudaStream_t st) {
  using Cfg = MmaCfg<DP, NR, TEAM, sizeof(T) == 4>;
  constexpr size_t ring = Cfg::WARPS * Cfg::WARP_BYTES;
  static_assert(ring + 8 * MU_ATTENTION_PAGED_MAX_REQUESTS <= 227 * 1024, "shared memory");
  static_assert(Cfg::CTAS_PER_SM * Cfg::WARPS <= MAX_WORKERS_PER_SM, "workspace");
  static_assert(2 * Cfg::CTAS_PER_SM * Cfg::WARPS * Cfg::R <= MAX_PART_ROWS_PER_SM, "workspace");
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(attention_paged_mma_kernel<T, DP, NR, TEAM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             ring + 8 * MU_ATTENTION_PAGED_MAX_REQUESTS) != cudaSuccess)
      return 2;
    once.set(1);
  }
  const int ctas = num_sms * Cfg::CTAS_PER_SM;
  a.rows_per_tile = Cfg::R;
  if (launch_behind(attention_paged_mma_kernel<T, DP, NR, TEAM>, ctas, Cfg::THREADS, ring + 8ull * a.B, chunks != nullptr, st, a))
    return 2;
  return launch_join<T>(a, JoinShare{ctas * Cfg::WARPS / TEAM, TEAM == 1 ? JOIN_WARPS : 1, 1}, chunks, num_sms, st);
}
template <typename T, int DP, int NR> int launch_mma(const PagedArgs &a, const PagedArgs *chunks, int num_sms, cudaStream_t st) {
  // Items (an upper bound) against warps: below an eighth every item would be cut into more than eight
  // pieces, and CTAs become the workers.
  const long long tiles = (1ll * a.n_tokens * a.G + 8 * NR - 1) / (8 * NR);
  const long long items = a.Hkv * (tiles > a.B ? tiles : a.B);
  if (items * 8 <= 1ll * num_sms * MmaCfg<DP, NR, 1, sizeof(T) == 4>::CTAS_PER_SM * MmaCfg<DP, NR, 1, sizeof(T) == 4>::WARPS)
    return launch_mma_team<T, DP, NR, 4>(a, chunks, num_sms, st);
  return launch_mma_team<T, DP, NR, 1>(a, chunks, num_sms, st);
}

template <typename T> int launch_by_dim(const PagedArgs &a, const PagedArgs *chunks, int num_sms, cudaStream_t st) {
  if (a.D % 16 != 0) {
    if (a.D % 4 != 0)
      return launch_simt_rows<T, 1, 8>(a, num_sms, st);
    return a.D <= 128 ? launch_simt_rows<T, 4, 1>(a, num_sms, st) : launch_simt_rows<T, 4, 2>(a, num_sms, st);
  }
  // 8 rows share every key read for single tokens (the group's heads), 16 where there are more
  const bool more = a.n_tokens > a.B || a.G > 8;
  if (a.D > 128)
    return launch_mma<T, 256, 1>(a, chunks, num_sms, st);
  if (a.D > 96)
    return more ? launch_mma<T, 128, 2>(a, chunks, num_sms, st) : launch_mma<T, 128, 1>(a, chunks, num_sms, st);
  if (a.D > 64)
    return more ? launch_mma<T, 96, 2>(a, chunks, num_sms, st) : launch_mma<T, 96, 1>(a, chunks, num_sms, st);
  if (a.D > 32)
    return more ? launch_mma<T, 64, 2>(a, chunks, num_sms, st) : launch_mma<T, 64, 1>(a, chunks, num_sms, st);
  return more ? launch_mma<T, 32, 2>(a, chunks, num_sms, st) : launch_mma<T, 32, 1>(a, chunks, num_sms, st);
}

// 0 ok, 1 dtype not implemented, 2 CUDA error
int launch_attention_paged(PagedArgs a, void *workspace, int dtype, int num_sms, cudaStream_t st) {
  unsigned char *w = static_cast<unsigned char *>(workspace);
  a.rows_from = 1, a.rows_to = INT_MAX;
  PagedArgs chunks = a;
  const bool tile = uses_tile_kernel(a.n_tokens, a.B, a.G, a.D, dtype);
  if (tile) {
    place_parts(chunks, w, 2ull * PAGED_TILE_ROWS * num_sms, num_sms);
    w += tile_part_bytes(num_sms, a.D);
    chunks.rows_from = TILE_KERNEL_ROWS, chunks.rows_per_tile = PAGED_TILE_ROWS;
    if (launch_attention_paged_tile(chunks, num_sms, st))
      return 2;
    a.rows_to = TILE_KERNEL_ROWS - 1;
  }
  place_parts(a, w, 1ull * MAX_PART_ROWS_PER_SM * num_sms, num_sms * MAX_WORKERS_PER_SM);
  if (dtype == F32)
    return launch_by_dim<float>(a, nullptr, num_sms, st);
  if (dtype == BF16)
    return launch_by_dim<__nv_bfloat16>(a, tile ? &chunks : nullptr, num_sms, st);
  return 1;
}

} // namespace mu

extern "C" {

int mu_set_error(mu_ctx *ctx, int code, const char *msg);
int mu_ctx_select_device(mu_ctx *ctx);
int mu_ctx_num_sms(const mu_ctx *ctx);
int *mu_ctx_status_ptr(mu_ctx *ctx);

size_t mu_attention_paged_workspace_bytes(const mu_ctx *ctx, int n_tokens, int B, int Hq, int Hkv, int D, int dtype) {
  if (!ctx || n_tokens <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0)
    return 0;
  return mu::paged_workspace_bytes(mu_ctx_num_sms(ctx), n_tokens, Hq / Hkv, D, dtype);
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
  if (num_pages == 0) // every page id is out of range: nothing is read, but addresses are formed
    k_cache = v_cache = workspace;
  mu::PagedArgs a{};
  a.q = q, a.out = out, a.q_ld = q_ld, a.out_ld = out_ld;
  a.kc = static_cast<const uint8_t *>(k_cache), a.vc = static_cast<const uint8_t *>(v_cache);
  a.ks = k_scale, a.vs = v_scale, a.table = block_table, a.table_stride = table_stride;
  a.query_start = query_start, a.seq_lens = seq_lens, a.B = B, a.n_tokens = n_tokens;
  a.Hq = Hq, a.Hkv = Hkv, a.G = Hq / Hkv, a.D = D, a.num_pages = num_pages, a.page_size = page_size;
  a.by_group = mu::FastDiv(a.G), a.by_page = mu::FastDiv(page_size);
  a.causal = causal != 0, a.status = mu_ctx_status_ptr(ctx);
  a.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(D)));
  if (mu::launch_attention_paged(a, workspace, dtype, mu_ctx_num_sms(ctx), static_cast<cudaStream_t>(stream)))
    return mu_set_error(ctx, MU_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
  return MU_OK;
}

} // extern "C"
