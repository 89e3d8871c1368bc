// Page bookkeeping of a paged KV cache and the write into its 8-bit pages.
//
// Layout: k_cache / v_cache [num_pages][Hkv][page_size][D] e4m3, k_scale / v_scale
// [num_pages][Hkv] float32; value = e4m3 * scale. Keys of one head inside one page are contiguous,
// so attention reads page_size * D bytes in a row. Slot of a token = page * page_size + offset.
//
// No counterpart in the reference (it has no KV cache); the argument checks, the latched device
// status and the asynchronous streams are those of the other entry points.
#include "../../include/munet_b200.h"
#include "common.h"
#include "ptx.cuh"
#include <climits>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace mu {

// ---- page map -----------------------------------------------------------------------------------
// One launch. Every CTA scans the request lengths itself (two prefix sums kept in shared memory: new
// tokens and new pages), which costs less than a second launch or a grid-wide barrier; the grid then
// shares out the new table entries and the tokens, each finding its request by binary search.
// Entries of the block table that are read (pages a request holds already) and those that are written
// (its new pages) never overlap, so no order between CTAs is needed. Latency throughout: 4.0 us for 64 requests that
// gain a token each, 6.0 us for 512 requests and 53,000 tokens (0.8 MB).
constexpr int PM_THREADS = 512;

struct PageMapArgs {
  const int *context_lens, *new_lens, *free_pages;
  int n_free;
  int *block_table;
  int table_stride, B, page_size, num_pages;
  int *query_start, *seq_lens, *slots, *positions;
  int n_slots;
  int *pages_taken;
  int *status;
};

// Index of the first entry of ends[0..n) that is > v (n when there is none).
__device__ __forceinline__ int upper_bound(const int *ends, int n, int v) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > v)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

struct ReqLens {
  int ctx, add, old_pages, new_pages;
  bool ok, fits;
};
// Lengths of one request; a negative one, or a sum beyond int32, counts as an empty request.
__device__ __forceinline__ ReqLens req_lens(const PageMapArgs &a, int r) {
  ReqLens q;
  q.ctx = a.context_lens[r], q.add = a.new_lens[r];
  const long long total = 1ll * q.ctx + q.add;
  q.ok = q.ctx >= 0 && q.add >= 0 && total <= INT_MAX;
  if (!q.ok)
    q.ctx = q.add = 0;
  const unsigned ps = a.page_size;
  const int have = static_cast<int>((static_cast<unsigned>(q.ctx) + ps - 1) / ps);
  const int want = static_cast<int>((static_cast<unsigned>(q.ctx) + static_cast<unsigned>(q.add) + ps - 1) / ps);
  q.fits = want <= a.table_stride;
  q.old_pages = min(have, a.table_stride);
  q.new_pages = min(want, a.table_stride) - q.old_pages;
  return q;
}

__global__ void __launch_bounds__(PM_THREADS) page_map_kernel(PageMapArgs a) {
  extern __shared__ int sm[];
  int *tok_end = sm, *page_end = sm + a.B; // inclusive prefix sums, saturated at INT_MAX
  __shared__ long long warp_tok[PM_THREADS / 32], warp_page[PM_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + PM_THREADS - 1) / PM_THREADS;
  const int r0 = min(tid * per, a.B), r1 = min(r0 + per, a.B);
  long long toks = 0, pages = 0;
  bool bad = false, full = false;
  for (int r = r0; r < r1; ++r) {
    const ReqLens q = req_lens(a, r);
    bad |= !q.ok, full |= !q.fits;
    toks += q.add, pages += q.new_pages;
    if (blockIdx.x == 0)
      a.seq_lens[r] = q.ctx + q.add;
  }
  long long st = toks, sp = pages;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long t = __shfl_up_sync(~0u, st, d), p = __shfl_up_sync(~0u, sp, d);
    if (lane >= d)
      st += t, sp += p;
  }
  if (lane == 31)
    warp_tok[warp] = st, warp_page[warp] = sp;
  __syncthreads();
  long long bt = st - toks, bp = sp - pages, all_tok = 0, all_page = 0;
#pragma unroll
  for (int w = 0; w < PM_THREADS / 32; ++w) {
    if (w < warp)
      bt += warp_tok[w], bp += warp_page[w];
    all_tok += warp_tok[w], all_page += warp_page[w];
  }
  for (int r = r0; r < r1; ++r) {
    const ReqLens q = req_lens(a, r);
    if (blockIdx.x == 0)
      a.query_start[r] = static_cast<int>(min(bt, 1ll * INT_MAX));
    bt += q.add, bp += q.new_pages;
    tok_end[r] = static_cast<int>(min(bt, 1ll * INT_MAX));
    page_end[r] = static_cast<int>(min(bp, 1ll * INT_MAX));
  }
  if (blockIdx.x == 0) {
    if (bad)
      atomicCAS(a.status, 0, MU_DEV_BAD_LENGTH);
    if (full || (tid == 0 && (all_tok > a.n_slots || all_page > a.n_free)))
      atomicCAS(a.status, 0, MU_DEV_NO_PAGE);
    if (tid == 0) {
      a.query_start[a.B] = static_cast<int>(min(all_tok, 1ll * INT_MAX));
      a.pages_taken[0] = static_cast<int>(min(all_page, 1ll * a.n_free));
    }
  }
  __syncthreads();

  const unsigned ps = a.page_size;
  const int stride = gridDim.x * PM_THREADS, first = blockIdx.x * PM_THREADS + tid;
  // new pages: entry j of the free list goes to the request whose range of new pages holds j
  const long long fresh = min(all_page, 1ll * INT_MAX - stride);
  for (int f = first; f < fresh; f += stride) {
    const int r = upper_bound(page_end, a.B, f);
    if (r >= a.B)
      break;
    const ReqLens q = req_lens(a, r);
    const int j = f - (r ? page_end[r - 1] : 0); // the sum before r is at most f, so it is not saturated
    int page = f < a.n_free ? a.free_pages[f] : -1;
    if (f < a.n_free && (page < 0 || page >= a.num_pages)) {
      atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
      page = -1;
    }
    a.block_table[1ll * r * a.table_stride + q.old_pages + j] = page;
  }
  // tokens: a page the request held before comes from its table, a new one from the free list
  const int limit = static_cast<int>(min(all_tok, 1ll * a.n_slots));
  for (long long tl = first; tl < a.n_slots; tl += stride) {
    const int t = static_cast<int>(tl);
    int slot = -1, pos = 0;
    if (t < limit) {
      const int r = upper_bound(tok_end, a.B, t);
      const ReqLens q = req_lens(a, r);
      pos = q.ctx + (t - (r ? tok_end[r - 1] : 0));
      const int pi = static_cast<int>(static_cast<unsigned>(pos) / ps);
      int page = -1;
      bool known = false;
      if (pi < q.old_pages) {
        page = a.block_table[1ll * r * a.table_stride + pi];
        known = true;
      } else if (pi < q.old_pages + q.new_pages) {
        const long long f = (r ? page_end[r - 1] : 0ll) + (pi - q.old_pages); // saturated: beyond any free list
        if (f < a.n_free)
          page = a.free_pages[f], known = true;
      }
      if (page >= 0 && page < a.num_pages)
        slot = static_cast<int>(static_cast<unsigned>(page) * ps + static_cast<unsigned>(pos) % ps);
      else if (known)
        atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

// 0 ok, 2 CUDA error
int launch_page_map(const PageMapArgs &a, int num_sms, cudaStream_t st) {
  const size_t smem = 2ull * sizeof(int) * a.B;
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(page_map_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(2 * sizeof(int) * MU_PAGE_MAP_MAX_REQUESTS)) != cudaSuccess)
      return 2;
    once.set(1);
  }
  long long blocks = (1ll * a.n_slots + PM_THREADS - 1) / PM_THREADS; // a new page holds a new token at least
  if (blocks > num_sms)
    blocks = num_sms;
  if (blocks < 1)
    blocks = 1;
  page_map_kernel<<<static_cast<unsigned>(blocks), PM_THREADS, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

// ---- write into the cache -----------------------------------------------------------------------
// Work unit: the run of consecutive new tokens that fall into one page, for one head of K or V. A team of
// threads finds the run's largest magnitude, derives the page's scale, requantises what the page held
// before if the scale grew, and stores the new rows. The rows stay in registers, as they came, between
// the two steps (64 elements per thread: a page of 64 x 128 for a team of 128), so HBM sees them once.
// Teams: a CTA where the tokens are many (prompts: one run per page); a warp, four heads to the CTA, where
// they are few (a decode step: every token is a run of its own, and a CTA would idle over 128 elements).
// Many tokens are bound by instructions: 64 prompts of up to 1024 tokens, 16 heads of 128 in bfloat16, take 62 us
// (240 MB: 3.9 TB/s). Few are latency, slot -> scale -> row -> store: 64 tokens 3.8 us, 15 us where every scale
// grows and the pages' earlier tokens are written again.
//
// Scale: the smallest power of two s >= 2^-64 with amax <= 448 s. e4m3 keeps its three mantissa bits
// at every magnitude, so a power of two loses nothing against amax/448 except range at the bottom,
// and growing it later is exact for everything above the subnormals.
constexpr int AP_THREADS = 128, AP_WARPS = AP_THREADS / 32;
constexpr int AP_REGS = 8;       // vectors of 8 elements a thread keeps
constexpr int AP_MAX_BLOCK = 64; // most tokens one CTA looks at for run starts

struct AppendArgs {
  const void *x[2]; // K, V
  long long ld;     // elements between tokens
  const int *slots;
  int n_tokens;
  uint8_t *cache[2];
  float *scale[2];
  int num_pages, page_size, H, D;
  FastDiv by_page;
  int block_tokens; // tokens per CTA
  int unit_blocks;  // CTAs that share a block of tokens
  unsigned dv, dv_magic; // vectors per row and ceil(2^32 / dv)
  int row_step, col_step; // rows and vectors that as many vectors as a team has threads make
  int *status;
};

// VE elements of a row as they are in memory: 8 (one or two 16-byte loads) or 1
template <typename T, int VE> struct RowVec {
  static constexpr int WORDS = VE == 8 ? 8 * sizeof(T) / 4 : 1;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (VE == 8) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
    } else {
      w[0] = __float_as_uint(static_cast<float>(*p));
    }
  }
  __device__ __forceinline__ void floats(float (&f)[VE]) const {
    if constexpr (VE == 8 && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        f[i] = __uint_as_float(w[i]);
    }
  }
};
// Largest magnitude of a vector as the bits of a float, infinities and NaN among them: two bfloat16 at a time.
template <typename T, int VE> __device__ __forceinline__ uint32_t amax_any(const RowVec<T, VE> &r, uint32_t m) {
  if constexpr (VE == 8 && sizeof(T) == 2) { // m: the largest of either half
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __vmaxu2(m, r.w[i] & 0x7fff7fffu);
  } else {
#pragma unroll
    for (int i = 0; i < RowVec<T, VE>::WORDS; ++i)
      m = max(m, r.w[i] & 0x7fffffffu);
  }
  return m;
}
template <typename T, int VE> __device__ __forceinline__ uint32_t amax_whole(uint32_t m) {
  return VE == 8 && sizeof(T) == 2 ? max(m & 0xffff0000u, m << 16) : m;
}
// largest finite magnitude, as bits (ordered like the values)
template <int VE> __device__ __forceinline__ uint32_t amax_bits(const float (&f)[VE], uint32_t m) {
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
    m = max(m, b < 0x7f800000u ? b : 0u);
  }
  return m;
}
// smallest power of two s >= 2^-64 with amax <= 448 s (448 = 1.75 * 2^8)
__device__ __forceinline__ float page_scale(uint32_t amax) {
  int e = static_cast<int>(amax >> 23) - 127; // subnormals end at the floor
  if ((amax & 0x7fffffu) > 0x600000u)         // mantissa above 1.75
    ++e;
  e = max(e - 8, -64);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
  return __half22float2(static_cast<__half2>(h));
}
// One rounding, from 64 bits: for scales that are no power of two (a cache that someone else filled). The
// value is rounded to e4m3's grid (three bits below its leading one, 2^-9 at least) in double; what comes out
// is exact in float and in the conversion.
__device__ __forceinline__ float on_e4m3_grid(double v) {
  if (!(fabs(v) < 1e6))
    return static_cast<float>(v); // saturates, or is NaN
  const int e = max(((__double2hiint(v) >> 20) & 0x7ff) - 1023, -6) - 3;
  return static_cast<float>(rint(v * __hiloint2double((1023 - e) << 20, 0)) * __hiloint2double((1023 + e) << 20, 0));
}
// Rows leave as v / s. A power of two's reciprocal is exact, so the product rounds once, in the conversion.
template <int VE> __device__ __forceinline__ void store_row_vec(uint8_t *dst, const float (&f)[VE], float inv) {
  if constexpr (VE == 8) {
    uint2 u;
    u.x = e4m3x2(f[0] * inv, f[1] * inv) | (e4m3x2(f[2] * inv, f[3] * inv) << 16);
    u.y = e4m3x2(f[4] * inv, f[5] * inv) | (e4m3x2(f[6] * inv, f[7] * inv) << 16);
    *reinterpret_cast<uint2 *>(dst) = u;
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      dst[i] = static_cast<uint8_t>(e4m3x2(f[i] * inv, 0.f) & 0xffu);
  }
}
// v / s for a scale that is no power of two, such that rounding it to e4m3's grid gives what the quotient itself
// would: in 64 bits, by the reciprocal; where that comes out next to a half step that v is an exact multiple of,
// the half step is the quotient. (A double division would be a call, and its registers the kernel's.)
__device__ __forceinline__ double exact_quotient(float v, float s, double recip) {
  const double q = v * recip;
  if (!(fabs(q) < 1e6))
    return q;
  const int e = max(((__double2hiint(q) >> 20) & 0x7ff) - 1023, -6) - 4; // half steps
  const double t = rint(q * __hiloint2double((1023 - e) << 20, 0)) * __hiloint2double((1023 + e) << 20, 0);
  return t * s == v ? t : q; // a half step has five bits: its product with s is exact
}
__device__ __forceinline__ double reciprocal(float s) {
  double r = 1.f / s;
  r = fma(r, fma(-r, static_cast<double>(s), 1.0), r);
  return fma(r, fma(-r, static_cast<double>(s), 1.0), r);
}
// What a page held, times held scale / new scale.
template <int TEAM> __device__ __forceinline__ void requantise(uint8_t *tile, int bytes, float held, float now, int tid) {
  // the new scale is a power of two, so q * f is exact in float for a held power of two and in double for any other
  const double f = held > 0.f ? static_cast<double>(held) * static_cast<double>(1.f / now) : 0.0;
  const bool pow2 = (__float_as_uint(held) & 0x7fffffu) == 0;
  const float ff = static_cast<float>(f);
  auto again = [&](uint32_t two) -> uint32_t {
    const float2 p = e4m3x2_to_float2(two);
    return pow2 ? e4m3x2(p.x * ff, p.y * ff) : e4m3x2(on_e4m3_grid(p.x * f), on_e4m3_grid(p.y * f));
  };
  auto word = [&](uint32_t u) { return again(u & 0xffffu) | (again(u >> 16) << 16); };
  // 16 bytes a thread; a lone warp has four loads under way (a page of 64 x 128 took it 32 us word by word)
  constexpr int E = TEAM == 32 ? 4 : 1;
  uint4 *w = reinterpret_cast<uint4 *>(tile);
  const int words = bytes / 16;
#pragma unroll 1
  for (int k = tid; k < words; k += E * TEAM) {
    uint4 u[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (k + e * TEAM < words)
        u[e] = w[k + e * TEAM];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (k + e * TEAM < words)
        w[k + e * TEAM] = make_uint4(word(u[e].x), word(u[e].y), word(u[e].z), word(u[e].w));
  }
#pragma unroll 1
  for (int k = (bytes & ~15) + tid; k < bytes; k += TEAM)
    tile[k] = static_cast<uint8_t>(again(tile[k]) & 0xffu);
}

// First set bit of `bits` at or after `from`, `n` if none below n.
__device__ __forceinline__ int next_bit(const uint32_t *bits, int from, int n) {
  for (int w = from >> 5; w * 32 < n; ++w) {
    uint32_t v = bits[w];
    if (w == from >> 5)
      v &= ~0u << (from & 31);
    if (v)
      return min(w * 32 + __ffs(v) - 1, n);
  }
  return n;
}

// New tokens of one page: the first one's place in the window, their number (its complement: out of order),
// the page, and the lowest offset in it.
struct __align__(16) Run {
  int i, n, page, low;
};

template <typename T, int VE, int TEAM>
__global__ void __launch_bounds__(AP_THREADS, VE == 8 ? (sizeof(T) == 2 ? (TEAM == 32 ? 4 : 8) : 4) : 4) kv_append_kernel(AppendArgs a) {
  // window of slots: the CTA's tokens and as many as one page holds after them
  extern __shared__ int sm[];
  const int token_block = blockIdx.x / a.unit_blocks, unit_block = blockIdx.x - token_block * a.unit_blocks;
  const int win = min(a.block_tokens + a.page_size, a.n_tokens - token_block * a.block_tokens);
  const int words = (a.block_tokens + a.page_size + 31) / 32;
  int *slot = sm;                                                             // [win]
  uint32_t *starts = reinterpret_cast<uint32_t *>(sm + a.block_tokens + a.page_size); // token begins a run (or none)
  uint32_t *disorder = starts + words;                                        // token continues a run at a lower offset
  __shared__ uint32_t red[AP_WARPS];
  __shared__ Run runs[AP_MAX_BLOCK];
  __shared__ int n_runs;
  const int t0 = token_block * a.block_tokens;
  const int ps = a.page_size, n_slots = a.num_pages * ps; // a slot fits 31 bits
  for (int i = threadIdx.x; i < words * 32; i += AP_THREADS) { // whole warps: the ballots need every lane
    int s = -1, before = -1;
    if (i < win) {
      s = a.slots[t0 + i];
      before = t0 + i > 0 ? a.slots[t0 + i - 1] : -1;
      if (s >= n_slots) {
        if (unit_block == 0)
          atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
        s = -1;
      }
      if (s < -1 && unit_block == 0)
        atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
      if (before >= n_slots)
        before = -1;
      slot[i] = s;
    }
    const bool same = s >= 0 && before >= 0 && a.by_page.div(s) == a.by_page.div(before);
    const uint32_t st = __ballot_sync(~0u, !same), di = __ballot_sync(~0u, same && s <= before);
    if ((threadIdx.x & 31) == 0)
      starts[i >> 5] = st, disorder[i >> 5] = di;
  }
  __syncthreads();
  // One thread finds the runs that begin among the CTA's tokens (by every thread: 70 us for 64 prompts, so 67).
  if (threadIdx.x == 0) {
    int found = 0;
#pragma unroll 1
    for (int i = next_bit(starts, 0, a.block_tokens); i < a.block_tokens && i < win;) {
      const int after = next_bit(starts, i + 1, win);
      if (slot[i] >= 0) {
        Run r;
        r.i = i, r.n = after - i, r.page = a.by_page.div(slot[i]);
        const int page0 = r.page * ps;
        r.low = slot[i] - page0;
        // A run in ascending order ends within the window. One that is out of order, or repeats a slot,
        // takes the slow walk below, token by token, so that the last write of a slot is the one that stays.
        if (next_bit(disorder, i + 1, after) < after || r.n > ps) {
          int j = i + 1;
          for (; t0 + j < a.n_tokens; ++j) {
            const int s = a.slots[t0 + j];
            if (s < 0 || s >= n_slots || a.by_page.div(s) != r.page)
              break;
            r.low = min(r.low, s - page0);
          }
          r.n = ~(j - i);
        }
        runs[found++] = r;
      }
      i = after;
    }
    n_runs = found;
  }
  __syncthreads();

  // this team's head of K or V
  const int tid = TEAM == AP_THREADS ? threadIdx.x : threadIdx.x & 31;
  const int unit = TEAM == AP_THREADS ? unit_block : unit_block * AP_WARPS + (threadIdx.x >> 5);
  if (unit >= 2 * a.H)
    return; // only whole warps of a CTA that meets no more at a barrier
  const int which = unit & 1, h = unit >> 1;
  const T *x = static_cast<const T *>(which ? a.x[1] : a.x[0]) + 1ll * h * a.D;
  auto team_sync = [] {
    if constexpr (TEAM == AP_THREADS)
      __syncthreads();
    else
      __syncwarp();
  };
  // row of vector v: exact for v < 2^18, dv <= 2^8
  auto row_of = [&](unsigned v) { return a.dv == 1 ? v : __umulhi(v, a.dv_magic); };
  for (int at_run = 0; at_run < n_runs; ++at_run) {
    const Run run = runs[at_run];
    const bool ordered = run.n >= 0;
    const int i = run.i, n = ordered ? run.n : ~run.n, page = run.page, page0 = page * ps, low = run.low;
    uint8_t *tile = (which ? a.cache[1] : a.cache[0]) + (1ull * page * a.H + h) * ps * a.D;
    float *scale = (which ? a.scale[1] : a.scale[0]) + 1ull * page * a.H + h;
    const float held = low > 0 ? *scale : 0.f;
    const T *rows = x + (1ll * t0 + i) * a.ld;

    // vector tid + k TEAM of the run is (row, col); the next one is a few rows further
    struct At {
      int row, col;
    };
    const int dv = a.dv;
    auto step = [&](At &at) {
      at.row += a.row_step, at.col += a.col_step;
      if (at.col >= dv)
        at.col -= dv, ++at.row;
    };
    const At begin{static_cast<int>(row_of(tid)), tid - static_cast<int>(row_of(tid)) * dv};

    RowVec<T, VE> keep[AP_REGS];
    uint32_t m = 0;
    At at = begin;
#pragma unroll
    for (int k = 0; k < AP_REGS; ++k, step(at))
      if (at.row < n)
        keep[k].load(rows + at.row * a.ld + at.col * VE);
    const At behind = at; // what the registers do not hold
    at = begin;
#pragma unroll
    for (int k = 0; k < AP_REGS; ++k, step(at))
      if (at.row < n)
        m = amax_any<T, VE>(keep[k], m);
#pragma unroll 1
    for (at = behind; at.row < n; step(at)) {
      RowVec<T, VE> r;
      r.load(rows + at.row * a.ld + at.col * VE);
      m = amax_any<T, VE>(r, m);
    }
    auto team_max = [&](uint32_t mine) {
      team_sync(); // the held scale has been read by all, and red[] is free
      mine = __reduce_max_sync(~0u, mine);
      if constexpr (TEAM == AP_THREADS) {
        if ((tid & 31) == 0)
          red[tid >> 5] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < AP_WARPS; ++w)
          mine = max(mine, red[w]);
      }
      return mine;
    };
    m = team_max(amax_whole<T, VE>(m));
    if (m >= 0x7f800000u) { // infinities or NaN: once more, without them
      m = 0;
#pragma unroll 1
      for (at = begin; at.row < n; step(at)) {
        RowVec<T, VE> r;
        float f[VE];
        r.load(rows + at.row * a.ld + at.col * VE);
        r.floats(f);
        m = amax_bits<VE>(f, m);
      }
      m = team_max(m);
    }
    const float now = fmaxf(held, page_scale(m));
    if (tid == 0)
      *scale = now;
    const bool fast = ordered && (__float_as_uint(now) & 0x7fffffu) == 0;
    if (fast) {
      const float inv = 1.f / now;
      at = begin;
#pragma unroll
      for (int k = 0; k < AP_REGS; ++k, step(at))
        if (at.row < n) {
          float f[VE];
          keep[k].floats(f);
          store_row_vec<VE>(tile + (slot[i + at.row] - page0) * a.D + at.col * VE, f, inv);
        }
#pragma unroll 1
      for (at = behind; at.row < n; step(at)) {
        RowVec<T, VE> r;
        float f[VE];
        r.load(rows + at.row * a.ld + at.col * VE);
        r.floats(f);
        store_row_vec<VE>(tile + (slot[i + at.row] - page0) * a.D + at.col * VE, f, inv);
      }
    }
    // the tokens before the new ones, low * D bytes from the tile's start: now that the rows' registers are free
    if (low > 0 && now > held)
      requantise<TEAM>(tile, low * a.D, held, now, tid);
    if (!fast) {
      const double recip = reciprocal(now);
#pragma unroll 1
      for (int j = 0; j < n; ++j) {
        team_sync(); // the requantised bytes and the token before are in place
        uint8_t *dst = tile + (a.slots[t0 + i + j] - page0) * a.D;
#pragma unroll 1
        for (int d = tid; d < a.D; d += TEAM)
          dst[d] = static_cast<uint8_t>(
              e4m3x2(on_e4m3_grid(exact_quotient(static_cast<float>(rows[j * a.ld + d]), now, recip)), 0.f) & 0xffu);
      }
    }
    team_sync(); // red[] is free again
  }
}

template <typename T> void launch_append_t(const AppendArgs &a, bool vec, int team, dim3 grid, size_t smem, cudaStream_t st) {
  if (team == 32) {
    if (vec)
      kv_append_kernel<T, 8, 32><<<grid, AP_THREADS, smem, st>>>(a);
    else
      kv_append_kernel<T, 1, 32><<<grid, AP_THREADS, smem, st>>>(a);
  } else {
    if (vec)
      kv_append_kernel<T, 8, AP_THREADS><<<grid, AP_THREADS, smem, st>>>(a);
    else
      kv_append_kernel<T, 1, AP_THREADS><<<grid, AP_THREADS, smem, st>>>(a);
  }
}

// 0 ok, 1 dtype not implemented, 2 CUDA error
int launch_kv_append(AppendArgs a, int dtype, int num_sms, cudaStream_t st) {
  if (dtype != F32 && dtype != BF16)
    return 1;
  const int es = dtype == F32 ? 4 : 2;
  bool vec = a.D % 8 == 0 && (a.ld * es) % 16 == 0;
  for (int i = 0; i < 2; ++i)
    vec = vec && (reinterpret_cast<uintptr_t>(a.x[i]) & 15u) == 0;
  a.dv = vec ? a.D / 8 : a.D;
  a.dv_magic = static_cast<unsigned>((0x100000000ull + a.dv - 1) / a.dv); // unused where dv is 1
  // Few tokens: one per CTA and a warp for each of four heads. Many: up to a page of tokens per CTA, whose
  // threads all work on one head; with one token per CTA most would find that no run begins there.
  const long long units = 2ll * a.H * a.n_tokens;
  const int team = units <= num_sms * 64ll ? 32 : AP_THREADS;
  a.row_step = team / a.dv, a.col_step = team % a.dv;
  long long tb = team == 32 ? 1 : units / (num_sms * 64ll);
  if (tb > AP_MAX_BLOCK)
    tb = AP_MAX_BLOCK;
  if (tb > a.page_size)
    tb = a.page_size;
  if (tb < 1)
    tb = 1;
  a.block_tokens = static_cast<int>(tb);
  const int span = a.block_tokens + a.page_size, words = (span + 31) / 32;
  const size_t smem = sizeof(int) * (span + 2ull * words);
  // The heads of one block of tokens are neighbours in the grid: their rows are neighbours in memory (256 bytes
  // a head, kilobytes between tokens), so DRAM pages are read while they are open.
  a.unit_blocks = team == 32 ? (2 * a.H + AP_WARPS - 1) / AP_WARPS : 2 * a.H;
  const long long blocks = (a.n_tokens + tb - 1) / tb;
  const dim3 grid(static_cast<unsigned>(blocks * a.unit_blocks));
  if (dtype == F32)
    launch_append_t<float>(a, vec, team, grid, smem, st);
  else
    launch_append_t<__nv_bfloat16>(a, vec, team, grid, smem, st);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}

} // namespace mu

extern "C" {

int mu_set_error(mu_ctx *ctx, int code, const char *msg);
int mu_ctx_select_device(mu_ctx *ctx);
int mu_ctx_num_sms(const mu_ctx *ctx);
int *mu_ctx_status_ptr(mu_ctx *ctx);

int mu_page_map(mu_ctx *ctx, const int32_t *context_lens, const int32_t *new_lens, const int32_t *free_pages,
                int n_free, int32_t *block_table, int table_stride, int B, int page_size, int num_pages,
                int32_t *query_start, int32_t *seq_lens, int32_t *slots, int32_t *positions, int n_slots,
                int32_t *pages_taken, void *stream) {
  if (!ctx)
    return MU_ERR_INVALID;
  if (B < 0 || n_free < 0 || n_slots < 0 || table_stride < 0 || page_size <= 0 || num_pages < 0)
    return mu_set_error(ctx, MU_ERR_INVALID, "page_map: negative size");
  if (B > MU_PAGE_MAP_MAX_REQUESTS)
    return mu_set_error(ctx, MU_ERR_SIZE, "page_map: more than MU_PAGE_MAP_MAX_REQUESTS requests");
  if (1ll * num_pages * page_size > INT_MAX)
    return mu_set_error(ctx, MU_ERR_SIZE, "page_map: num_pages * page_size does not fit a 32-bit slot");
  if (!query_start || !pages_taken || (B > 0 && (!context_lens || !new_lens || !seq_lens)) ||
      (B > 0 && table_stride > 0 && !block_table) || (n_free > 0 && !free_pages) ||
      (n_slots > 0 && (!slots || !positions)))
    return mu_set_error(ctx, MU_ERR_INVALID, "page_map: null pointer");
  if (mu_ctx_select_device(ctx) != MU_OK)
    return mu_set_error(ctx, MU_ERR_CUDA, "page_map: cannot select device");
  const mu::PageMapArgs a{context_lens, new_lens, free_pages, n_free, block_table, table_stride, B, page_size,
                          num_pages, query_start, seq_lens, slots, positions, n_slots, pages_taken,
                          mu_ctx_status_ptr(ctx)};
  if (mu::launch_page_map(a, mu_ctx_num_sms(ctx), static_cast<cudaStream_t>(stream)))
    return mu_set_error(ctx, MU_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
  return MU_OK;
}

int mu_kv_cache_append(mu_ctx *ctx, const void *k, const void *v, long long ld, const int32_t *slots,
                       int n_tokens, void *k_cache, void *v_cache, float *k_scale, float *v_scale,
                       int num_pages, int page_size, int Hkv, int D, int dtype, void *stream) {
  if (!ctx)
    return MU_ERR_INVALID;
  if (n_tokens < 0 || num_pages < 0 || Hkv <= 0 || D <= 0 || page_size <= 0)
    return mu_set_error(ctx, MU_ERR_INVALID, "kv_cache_append: bad dimensions");
  if (page_size % 16 != 0 || page_size > 1024 || D > 256 || Hkv > 16384)
    return mu_set_error(ctx, MU_ERR_UNSUPPORTED, "kv_cache_append: page size a multiple of 16 up to 1024, head size "
                        "up to 256, at most 16384 heads");
  if (dtype != MU_F32 && dtype != MU_BF16)
    return mu_set_error(ctx, MU_ERR_UNSUPPORTED, "kv_cache_append: dtype not implemented (float32, bfloat16)");
  if (ld < 1ll * Hkv * D)
    return mu_set_error(ctx, MU_ERR_INVALID, "kv_cache_append: row stride below Hkv * D");
  if (1ll * num_pages * page_size > INT_MAX)
    return mu_set_error(ctx, MU_ERR_SIZE, "kv_cache_append: num_pages * page_size does not fit a 32-bit slot");
  if ((n_tokens / 16 + 1ll) * 2 * Hkv > INT_MAX)
    return mu_set_error(ctx, MU_ERR_SIZE, "kv_cache_append: tokens x heads beyond one launch");
  if (n_tokens == 0)
    return MU_OK;
  if (!k || !v || !slots || !k_cache || !v_cache || !k_scale || !v_scale)
    return mu_set_error(ctx, MU_ERR_INVALID, "kv_cache_append: null pointer");
  if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15u)
    return mu_set_error(ctx, MU_ERR_INVALID, "kv_cache_append: the caches must be 16-byte aligned");
  if (mu_ctx_select_device(ctx) != MU_OK)
    return mu_set_error(ctx, MU_ERR_CUDA, "kv_cache_append: cannot select device");
  mu::AppendArgs a{};
  a.x[0] = k, a.x[1] = v, a.ld = ld, a.slots = slots, a.n_tokens = n_tokens;
  a.cache[0] = static_cast<uint8_t *>(k_cache), a.cache[1] = static_cast<uint8_t *>(v_cache);
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.num_pages = num_pages, a.page_size = page_size, a.H = Hkv, a.D = D, a.status = mu_ctx_status_ptr(ctx);
  a.by_page = mu::FastDiv(page_size);
  if (mu::launch_kv_append(a, dtype, mu_ctx_num_sms(ctx), static_cast<cudaStream_t>(stream)))
    return mu_set_error(ctx, MU_ERR_CUDA, cudaGetErrorString(cudaGetLastError()));
  return MU_OK;
}

} // extern "C"
