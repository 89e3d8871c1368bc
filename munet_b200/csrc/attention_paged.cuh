// Shared pieces of the kernels that attend over the paged e4m3 cache (attention_paged.cu: the cache's
// reader for few rows per request; attention_paged_tile.cu: prompt chunks).
#pragma once
#include "common.h"
#include "ptx.cuh"
#include <climits>
#include <cuda_fp16.h>

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
  FastDiv by_group, by_page;
  float scale_log2; // log2(e) / sqrt(D)
  struct SplitItem *items; // by the worker that holds the first chunk
  int2 *notes;             // per worker: rows of the split item it begins (0: none), worker that began the
                           // item its first segment continues (-1: none)
  float2 *part_ml;
  float *part_o;
  int rows_per_tile; // stride of the partial results
  int rows_from, rows_to; // requests with this many rows (tokens x heads of a group), inclusive, are this kernel's
  int *status;
};

// A (request, head, row tile) whose chunks went to more than one worker; entry w belongs to the worker
// that holds its first chunk. Its later pieces are the first segments of workers w+1 .. last.
struct SplitItem {
  int first_slot, last, row0, n_rows, q0, head;
};

constexpr int START_UNITS = 3; // what beginning an item counts for, in chunks (1: 69.3 us, 2: 67.3, 3: 66.3 for 64 requests)

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
  if (s.nq * a.G < a.rows_from || s.nq * a.G > a.rows_to)
    s.nq = 0;
  // what the table can address; key numbers a few tiles behind the last one must not leave 31 bits either
  const long long room = min(1ll * a.table_stride * a.page_size, 1ll * INT_MAX - 65536);
  s.seen = s.len;
  if (s.nq > 0 && s.len > room) {
    atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
    s.seen = static_cast<int>(room);
  }
  return s;
}
// Keys row `row` of a request may see.
__device__ __forceinline__ int row_limit(const PagedArgs &a, const Seq &s, int row) {
  if (row >= s.nq * a.G)
    return 0;
  if (!a.causal)
    return s.seen;
  return max(0, min(s.seen, s.len - s.nq + a.by_group.div(row) + 1));
}

struct Segment {
  int b, head, n_rows, row0; // request, KV head, rows of the tile that exist, first of them
  int chunk0, chunks;        // range of this worker
  int slot;                  // -1: complete
};

// Unit counts hardly ever need 64 bits, and a 64-bit division costs a hundred instructions.
__device__ __forceinline__ long long div64(long long x, long long d) {
  if (((x | d) >> 32) == 0)
    return static_cast<unsigned>(x) / static_cast<unsigned>(d);
  return x / d;
}
__device__ __forceinline__ long long div_rem(long long x, int d, int &rem) {
  const long long q = div64(x, d);
  rem = static_cast<int>(x - q * d);
  return q;
}

__device__ __forceinline__ void store_out(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float load_in(const float *p) { return *p; }
__device__ __forceinline__ float load_in(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
// weight of a piece whose running maximum is m where the whole's is M
__device__ __forceinline__ float rel_weight(float m, float M) { return M == -INFINITY ? 1.f : ex2_approx(m - M); }

// attention_paged_tile.cu: rows a tile of it holds, requests its prefix sums have room for beside the operands
constexpr int PAGED_TILE_ROWS = 256, MU_PAGED_TILE_MAX_REQUESTS = 3500;
int launch_attention_paged_tile(const PagedArgs &a, int num_sms, cudaStream_t st);

// e4m3 pairs to fp16 pairs: exact
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
__device__ __forceinline__ bool has_nan_e4m3(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

} // namespace mu
