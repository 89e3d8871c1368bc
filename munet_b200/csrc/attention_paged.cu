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

// ---- tensor-core kernel: bfloat16 queries, head size 64 or 128 -------------------------------------
// Bound by reading the cache. Sixteen rows (tokens x heads of the group) share every key. Each of the
// four warps works alone on every fourth tile of 32 keys: it copies the tile's K and V bytes into its
// own ring in shared memory (cp.async, 16 bytes a lane; MMA_STAGES tiles of 64 D bytes in flight), turns
// them into fp16 in registers and multiplies with mma.m16n8k16. Nothing but the end of a segment
// synchronises the CTA.
//
// Numbers: e4m3 is exact in fp16. A query row is scaled by a power of two to at most 2^15, which keeps a
// bfloat16 mantissa exact. A page's K scale multiplies its fp32 scores. Its V scale goes into the weight:
// with t = s + log2(vs), weights are 2^(t - max t + 12) in fp16 (2^-12 of them lies above the fp16
// subnormals, so a page of small values that matters keeps its bits), and the softmax sum takes
// w / vs back out in fp32.
//
// Both products may permute what they sum over, so fragments are read straight from the bytes: in q.k lane
// c of a quad owns dimensions [c D/4, (c+1) D/4); in p.v lane group g owns dimensions [g D/8, (g+1) D/8).
// 16-byte chunks are XOR-swizzled by the key's row so that those reads meet no bank twice.
constexpr int MMA_WARPS = 4, MMA_THREADS = 32 * MMA_WARPS, MMA_ROWS = 16, MMA_TILE = 32;
constexpr int MMA_CTAS_PER_SM = 2;
template <int D> struct MmaCfg {
  static constexpr int STAGES = D == 128 ? 3 : 6;
  static constexpr int TILE_BYTES = MMA_TILE * D;           // of K, and of V
  static constexpr int WARP_BYTES = STAGES * 2 * TILE_BYTES; // 24 KB
  static_assert(WARP_BYTES >= MMA_ROWS * D * 4, "a warp's ring also carries its rows at the end");
};

__device__ __forceinline__ uint32_t f16x2_of_e4m3_lo(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3_hi(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(d) : "r"(w));
  return d;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes into shared memory, or 16 zero bytes
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// byte offset of 16-byte chunk `chunk` of row `row` in a tile
template <int D> __device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
  if constexpr (D == 128)
    return row * 128 + ((chunk ^ (row & 7)) << 4);
  else
    return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
__device__ __forceinline__ bool has_nan_e4m3(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

// Page of a half tile (16 keys never leave a page) and its scales, one per lane.
struct HalfPage {
  int page; // -1: none
  float ks, lv, iv; // K scale, log2 and reciprocal of the V scale
};
__device__ __forceinline__ HalfPage load_half(const PagedArgs &a, const Segment &g, int key, int end) {
  HalfPage h;
  h.page = -1, h.ks = 0.f, h.lv = -INFINITY, h.iv = 0.f;
  if (key < end) {
    const int page = a.table[1ll * g.b * a.table_stride + static_cast<unsigned>(key) / static_cast<unsigned>(a.page_size)];
    if (page >= 0 && page < a.num_pages) {
      const long long t = 1ll * page * a.Hkv + g.head;
      const float vs = fmaxf(a.vs[t], 0x1p-64f);
      h.page = page, h.ks = a.ks[t], h.lv = log2f(vs), h.iv = 1.f / vs;
    } else {
      atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
    }
  }
  return h;
}

template <int D> __global__ void __launch_bounds__(MMA_THREADS, MMA_CTAS_PER_SM) attention_paged_mma_kernel(PagedArgs a) {
  using Cfg = MmaCfg<D>;
  constexpr int S = Cfg::STAGES, KW = D / 16, NT = D / 8; // k-steps of q.k = 32-bit words a lane reads per key; n-tiles of p.v
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ long long warp_sum[MMA_WARPS];
  __shared__ float2 ml_s[MMA_WARPS][MMA_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, grp = lane >> 2, quad = lane & 3;
  unsigned char *ring = smem_raw + warp * Cfg::WARP_BYTES;
  long long *upto = reinterpret_cast<long long *>(smem_raw + MMA_WARPS * Cfg::WARP_BYTES);
  const uint32_t ring_u32 = smem_u32(ring);

  if (tid == 0)
    a.items[blockIdx.x].used = 0;
  const long long total = scan_units<MMA_THREADS, MMA_ROWS>(a, upto, warp_sum);
  if (total == 0)
    return;
  Walk walk(total, blockIdx.x, gridDim.x);
  Segment g;
  Seq s;
  const unsigned ps = a.page_size;
  while (walk.next<MMA_ROWS>(a, upto, g, s)) {
    // limits: least over the tile's rows, most over them, and this lane's two rows
    const int least = row_limit(a, s, g.row0), most = row_limit(a, s, g.row0 + g.n_rows - 1);
    const int lim0 = row_limit(a, s, g.row0 + grp), lim1 = row_limit(a, s, g.row0 + grp + 8);
    const int first = g.chunk0 * CHUNK + warp * MMA_TILE, end = min(most, (g.chunk0 + g.chunks) * CHUNK);
    const int tiles = end > first ? (end - first + CHUNK - 1) / CHUNK : 0; // this warp's, CHUNK apart
    auto half_key = [&](int batch) { return first + (batch * 16 + (lane >> 1)) * CHUNK + (lane & 1) * 16; };
    HalfPage cur = load_half(a, g, half_key(0), end), nxt = load_half(a, g, half_key(1), end);

    auto issue = [&](int i, const HalfPage &hp) {
      if (i < tiles) {
        const uint32_t st = ring_u32 + (i % S) * 2 * Cfg::TILE_BYTES;
        const int key0 = first + i * CHUNK;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int page = __shfl_sync(~0u, hp.page, (i & 15) * 2 + hf);
          const int key = key0 + 16 * hf, live = page >= 0 ? s.seen - key : 0; // rows behind it hold anything
          const unsigned in_page = static_cast<unsigned>(key) % ps;
          const long long off = page >= 0 ? ((1ll * page * a.Hkv + g.head) * ps + in_page) * D + lane * 16 : 0;
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int idx = lane + 32 * j, row = idx / (D / 16), chunk = idx % (D / 16);
            const uint32_t at = tile_at<D>(hf * 16 + row, chunk);
            const bool real = row < live;
            const long long o = real ? off + 512 * j : 0;
            cp_async16(st + at, a.kc + o, real);
            cp_async16(st + Cfg::TILE_BYTES + at, a.vc + o, real);
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
      issue(i, cur);

    // queries: fp16 fragments and each row's factor back
    uint32_t qf[KW][4];
    float fac[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float v[D / 4];
      const bool live = grp + 8 * r < g.n_rows;
      const long long row = g.row0 + grp + 8 * r;
      const __nv_bfloat16 *qp = static_cast<const __nv_bfloat16 *>(a.q) +
                                (live ? (s.q0 + row / a.G) * a.q_ld + (1ll * g.head * a.G + row % a.G) * D + quad * (D / 4) : 0);
      if ((reinterpret_cast<uintptr_t>(qp) & 15u) == 0 && live) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 u = *(reinterpret_cast<const uint4 *>(qp) + i);
          v[8 * i] = bf16_lo(u.x), v[8 * i + 1] = bf16_hi(u.x), v[8 * i + 2] = bf16_lo(u.y), v[8 * i + 3] = bf16_hi(u.y);
          v[8 * i + 4] = bf16_lo(u.z), v[8 * i + 5] = bf16_hi(u.z), v[8 * i + 6] = bf16_lo(u.w), v[8 * i + 7] = bf16_hi(u.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i)
          v[i] = live ? __bfloat162float(qp[i]) : 0.f;
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 4; ++i)
        top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(~0u, top, 1));
      top = max(top, __shfl_xor_sync(~0u, top, 2));
      const int e = min(max(static_cast<int>(top >> 23) - 127 - 14, -100), 113);
      const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      fac[r] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        qf[i][r] = f16x2(v[4 * i] * f, v[4 * i + 1] * f);
        qf[i][r + 2] = f16x2(v[4 * i + 2] * f, v[4 * i + 3] * f);
      }
    }

    float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
      o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    for (int i = 0; i < tiles; ++i) {
      if ((i & 15) == 0 && i > 0)
        cur = nxt, nxt = load_half(a, g, half_key((i >> 4) + 1), end);
      issue(i + S - 1, ((i + S - 1) >> 4) == (i >> 4) ? cur : nxt);
      cp_async_wait<S - 1>();
      __syncwarp();
      const unsigned char *kt = ring + (i % S) * 2 * Cfg::TILE_BYTES, *vt = kt + Cfg::TILE_BYTES;
      const int key0 = first + i * CHUNK;

      float sc[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
        sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
        uint32_t w[KW];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint4 u = *reinterpret_cast<const uint4 *>(kt + tile_at<D>(nt * 8 + grp, quad * (D / 64) + c));
          w[4 * c] = u.x, w[4 * c + 1] = u.y, w[4 * c + 2] = u.z, w[4 * c + 3] = u.w;
        }
#pragma unroll
        for (int k = 0; k < KW; ++k)
          mma_f16(sc[nt], qf[k], f16x2_of_e4m3_lo(w[k]), f16x2_of_e4m3_hi(w[k]));
      }
      float iv[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int src = (i & 15) * 2 + hf;
        const float ks = __shfl_sync(~0u, cur.ks, src), lv = __shfl_sync(~0u, cur.lv, src);
        iv[hf] = __shfl_sync(~0u, cur.iv, src);
#pragma unroll
        for (int nt = 2 * hf; nt < 2 * hf + 2; ++nt) {
          sc[nt][0] = fmaf(sc[nt][0], ks * fac[0], lv), sc[nt][1] = fmaf(sc[nt][1], ks * fac[0], lv);
          sc[nt][2] = fmaf(sc[nt][2], ks * fac[1], lv), sc[nt][3] = fmaf(sc[nt][3], ks * fac[1], lv);
        }
      }
      const bool edge = key0 + MMA_TILE > least;
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + nt * 8 + quad * 2 + e;
            if (key >= lim0)
              sc[nt][e] = -INFINITY;
            if (key >= lim1)
              sc[nt][2 + e] = -INFINITY;
          }
      }
      float t0 = m0, t1 = m1;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
        t0 = fmaxf(t0, fmaxf(sc[nt][0], sc[nt][1])), t1 = fmaxf(t1, fmaxf(sc[nt][2], sc[nt][3]));
      t0 = fmaxf(t0, __shfl_xor_sync(~0u, t0, 1)), t1 = fmaxf(t1, __shfl_xor_sync(~0u, t1, 1));
      t0 = fmaxf(t0, __shfl_xor_sync(~0u, t0, 2)), t1 = fmaxf(t1, __shfl_xor_sync(~0u, t1, 2));
      const float ref0 = t0 == -INFINITY ? 0.f : t0 - 12.f, ref1 = t1 == -INFINITY ? 0.f : t1 - 12.f;
      if (__any_sync(~0u, t0 != m0 || t1 != m1)) {
        const float f0 = m0 == -INFINITY ? 0.f : ex2_approx(m0 - t0), f1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - t1);
        l0 *= f0, l1 *= f1;
#pragma unroll
        for (int j = 0; j < NT; ++j)
          o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
        m0 = t0, m1 = t1;
      }
      uint32_t pf[2][4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float (&x)[4] = sc[2 * hf + n];
          x[0] = ex2_approx(x[0] - ref0), x[1] = ex2_approx(x[1] - ref0);
          x[2] = ex2_approx(x[2] - ref1), x[3] = ex2_approx(x[3] - ref1);
          sum0 += x[0] + x[1], sum1 += x[2] + x[3];
          pf[hf][2 * n] = f16x2(x[0], x[1]), pf[hf][2 * n + 1] = f16x2(x[2], x[3]);
        }
        l0 = fmaf(sum0, iv[hf], l0), l1 = fmaf(sum1, iv[hf], l1);
      }

#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        constexpr int VW = D / 32; // 32-bit words a lane reads per key
        uint32_t w[4][VW];         // keys 2 quad, 2 quad + 1, and both + 8
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = hf * 16 + 2 * quad + (r & 1) + 8 * (r >> 1);
          if constexpr (D == 128) {
            const uint4 u = *reinterpret_cast<const uint4 *>(vt + tile_at<D>(row, grp));
            w[r][0] = u.x, w[r][1] = u.y, w[r][2] = u.z, w[r][3] = u.w;
          } else {
            const uint2 u = *reinterpret_cast<const uint2 *>(vt + tile_at<D>(row, grp >> 1) + (grp & 1) * 8);
            w[r][0] = u.x, w[r][1] = u.y;
          }
        }
        auto product = [&](float (&c)[4], const uint32_t (&p)[4], const uint32_t (&x)[4][VW], int j) {
          const uint32_t sel = j & 2 ? 0x7362 : 0x5140; // bytes of two keys side by side, two dimensions
          const uint32_t b0 = __byte_perm(x[0][j >> 2], x[1][j >> 2], sel), b1 = __byte_perm(x[2][j >> 2], x[3][j >> 2], sel);
          if (j & 1)
            mma_f16(c, p, f16x2_of_e4m3_hi(b0), f16x2_of_e4m3_hi(b1));
          else
            mma_f16(c, p, f16x2_of_e4m3_lo(b0), f16x2_of_e4m3_lo(b1));
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
          for (int j = 0; j < NT; ++j)
            product(o[j], pf[hf], w, j);
        } else {
          // A NaN among keys that some rows may not see: zero weights would not keep it out, so the keys go
          // one at a time and a row takes only those it sees.
#pragma unroll 1
          for (int t = 0; t < 16; ++t) {
            const int key = key0 + hf * 16 + t;
            uint32_t x[4][VW], p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool mine = t == 2 * quad + (r & 1) + 8 * (r >> 1);
#pragma unroll
              for (int q = 0; q < VW; ++q)
                x[r][q] = mine ? w[r][q] : 0u;
            }
            const uint32_t keep = (t & 7) >> 1 == quad ? (t & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              p[r] = (r >> 1) == (t >> 3) ? pf[hf][r] & keep : 0u;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              product(c, p, x, j);
              if (key < lim0)
                o[j][0] += c[0], o[j][1] += c[1];
              if (key < lim1)
                o[j][2] += c[2], o[j][3] += c[3];
            }
          }
        }
      }
      __syncwarp(); // the stage may be overwritten
    }
    cp_async_wait<0>();
    __syncwarp();

    // join the warps: every ring now carries its warp's rows
    l0 += __shfl_xor_sync(~0u, l0, 1), l1 += __shfl_xor_sync(~0u, l1, 1);
    l0 += __shfl_xor_sync(~0u, l0, 2), l1 += __shfl_xor_sync(~0u, l1, 2);
    if (quad == 0)
      ml_s[warp][grp] = make_float2(m0 - 12.f, l0), ml_s[warp][grp + 8] = make_float2(m1 - 12.f, l1);
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (grp + 8 * r < g.n_rows) {
        float *p = mine + (grp + 8 * r) * D + quad * (D / 4);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int j = 0; j < NT; j += 4)
            *reinterpret_cast<float4 *>(p + e * NT + j) =
                make_float4(o[j][2 * r + e], o[j + 1][2 * r + e], o[j + 2][2 * r + e], o[j + 3][2 * r + e]);
      }
    __syncthreads();
    for (int e = tid; e < g.n_rows * D; e += MMA_THREADS) {
      const int r = e / D, d = e % D;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < MMA_WARPS; ++w)
        M = fmaxf(M, ml_s[w][r].x);
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < MMA_WARPS; ++w) {
        const float f = rel_weight(ml_s[w][r].x, M);
        sum = fmaf(f, ml_s[w][r].y, sum);
        x = fmaf(f, reinterpret_cast<const float *>(smem_raw + w * Cfg::WARP_BYTES)[e], x);
      }
      if (g.slot < 0) {
        const long long row = g.row0 + r;
        store_out(static_cast<__nv_bfloat16 *>(a.out) + (s.q0 + row / a.G) * a.out_ld +
                      (1ll * g.head * a.G + row % a.G) * D + d,
                  sum == 0.f ? 0.f : x / sum);
      } else {
        const long long pr = 1ll * g.slot * a.rows_per_tile + r;
        a.part_o[pr * D + d] = x;
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

template <int D> int launch_mma(PagedArgs a, int num_sms, cudaStream_t st) {
  const size_t smem = MMA_WARPS * MmaCfg<D>::WARP_BYTES + 8ull * a.B;
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(attention_paged_mma_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             MMA_WARPS * MmaCfg<D>::WARP_BYTES + 8 * MU_ATTENTION_PAGED_MAX_REQUESTS) != cudaSuccess)
      return 2;
    once.set(1);
  }
  const int ctas = num_sms * MMA_CTAS_PER_SM;
  a.rows_per_tile = MMA_ROWS;
  attention_paged_mma_kernel<D><<<ctas, MMA_THREADS, smem, st>>>(a);
  if (cudaGetLastError() != cudaSuccess)
    return 2;
  return launch_join<__nv_bfloat16>(a, ctas, st);
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
  if (dtype == BF16 && a.D == 128)
    return launch_mma<128>(a, num_sms, st);
  if (dtype == BF16 && a.D == 64)
    return launch_mma<64>(a, num_sms, st);
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
