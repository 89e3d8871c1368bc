// Prompt chunks over the paged e4m3 cache: the tensor-core form of attention_paged.cu for requests with
// many rows (new tokens x query heads of a KV head), bfloat16, head size 64 or 128.
//
// Bound by the softmax in front of the tensor pipe: eight requests of up to 8192 keys with chunks of up to 2048 new
// tokens, 16 query and 4 KV heads of 128, take 691 us with the join (587 TFLOP/s; 730 between changes of work, which
// cost 11 us each); with heads of 64, 587 us (346 TFLOP/s: as many weights for half the products). Persistent, one CTA per SM, 16 warps:
//   warp 0      issues every tcgen05.mma (fp16 operands, fp32 accumulators in tensor memory)
//   warps 1-7   bring keys and values in: e4m3 bytes from their pages, turned into fp16 (exact) and
//               written where a TMA with 128-byte swizzle would have put them
//   warps 8-15  the softmax of query tiles A and B (128 rows each, one thread per row), as in the
//               prompt kernel of attention_tcgen05.cu: S in tensor memory, P written back over it as
//               fp16, O rescaled in place only when a row's maximum grew by more than 2^8
// A and B share every key tile of 128. Rows are (token, head) pairs, heads of a group next to each other.
//
// Scales as in attention_paged.cu: queries are scaled per row by a power of two, a page's K scale
// multiplies its scores, log2 of its V scale joins the exponent, and its reciprocal the softmax sum. A page
// holds whole groups of 16 keys, so these are constants per 16 columns.
//
// Work split: units of 8 keys, with the number that a causal row tile sees as a linear function of the
// tile, so that the prefix sum has a closed form; CTAs take equal shares and leave pieces where a share
// ends inside an item, which the join kernel adds up.
#include "attention_paged.cuh"
#include <cmath>
#include <type_traits>

namespace mu {

constexpr int PT_BQ = 128, PT_BK = 128, PT_ROWS = 2 * PT_BQ; // a row tile is the pair A, B
constexpr int PT_LOADERS = 7, PT_THREADS = 32 * (1 + PT_LOADERS + 8);
constexpr int PT_UNIT = 8, PT_START = 112; // keys of a unit; units that beginning an item counts for: seven key tiles
                                           // (16 units: 823 us for the mixed chunks above, 48: 770, 80: 717, 128: 712;
                                           // measured at head size 128 only)
constexpr int PT_SLOTS = 4;               // key tiles whose page scales are kept
constexpr float PT_W_EXP = 7.f;           // a row's reference weight is 2^7: with the 2^8 the maximum may lead, 2^15

template <int D> struct PtCfg {
  static constexpr int Q_BYTES = PT_BQ * D * 2, K_BYTES = PT_BK * D * 2, DB = D / 64;
  static constexpr int SMEM = 2 * Q_BYTES + 4 * K_BYTES; // Q_A, Q_B, two K and two V tiles
  static constexpr int BARS = 28;
  static constexpr int TAIL = BARS * 8 + PT_SLOTS * 8 * 16 + PT_SLOTS * 32 + 16;
};

// Byte of 16-byte word `word` of row `row` of a query tile: blocks of 64 dimensions, 128 bytes a row, swizzled. Queries
// and the output that is staged in their place both go through it, so a warp only ever touches its own rows' bytes and
// needs no barrier with the others of its tile between an output and the next work's queries.
__host__ __device__ constexpr int q_word(int row, int word) {
  return (word >> 3) * (PT_BQ * 128) + row * 128 + (((word & 7) ^ (row & 7)) << 4);
}
template <int D> constexpr bool rows_apart() { // within the tile, and in their own row's 128 bytes of each block
  for (int row = 0; row < PT_BQ; ++row)
    for (int word = 0; word < D / 8; ++word)
      if (q_word(row, word) < 0 || q_word(row, word) + 16 > PtCfg<D>::Q_BYTES || q_word(row, word) / 128 % PT_BQ != row)
        return false;
  return true;
}
static_assert(rows_apart<64>() && rows_apart<128>(), "rows of a query tile share bytes");

// Row tile costs of one request: tile t counts first + t * slope units, no fewer than the keys it sees / 8.
struct TileCosts {
  int tiles, slope;
  long long first, head; // of all tiles of one KV head
  __device__ __forceinline__ long long upto(int t) const { return t * first + static_cast<long long>(t) * (t - 1) / 2 * slope; }
};
__device__ __forceinline__ TileCosts tile_costs(const PagedArgs &a, const Seq &s) {
  TileCosts c;
  const int rows = s.nq * a.G;
  c.tiles = (rows + PT_ROWS - 1) / PT_ROWS;
  const int tokens = a.by_group.div(PT_ROWS - 1) + 2; // that a tile's rows can span, and one
  c.slope = a.causal ? (tokens + PT_UNIT - 1) / PT_UNIT : 0;
  const long long keys = a.causal ? 1ll * max(s.len - s.nq, 0) + tokens : s.seen;
  c.first = PT_START + (keys + PT_UNIT - 1) / PT_UNIT + 1;
  c.head = c.upto(c.tiles);
  return c;
}
__device__ __forceinline__ int tile_chunks(const PagedArgs &a, const Seq &s, int row0) {
  const int last = min(row0 + PT_ROWS, s.nq * a.G) - 1;
  return max(1, (row_limit(a, s, last) + PT_BK - 1) / PT_BK);
}

struct TileWalk {
  long long u, end, total;
  int workers, me, b;
  bool first;
  __device__ __forceinline__ TileWalk(long long total_, int me_, int grid) : total(total_), me(me_), b(0), first(true) {
    // several chunks to a share (16 units each)
    workers = static_cast<int>(min(static_cast<long long>(grid), max(1ll, total / 64)));
    u = end = 0;
    if (me < workers) {
      int rest;
      const long long each = div_rem(total, workers, rest);
      u = each * me + static_cast<unsigned>(rest * me) / static_cast<unsigned>(workers);
      end = each * (me + 1) + static_cast<unsigned>(rest * (me + 1)) / static_cast<unsigned>(workers);
    }
  }
  __device__ __forceinline__ int owner(long long x) const {
    return static_cast<int>(div64((x + 1) * workers - 1, total));
  }
  __device__ __forceinline__ bool next(const PagedArgs &a, const long long *upto, Segment &g, Seq &s, bool leader) {
    for (;;) {
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
      const TileCosts c = tile_costs(a, s);
      const long long local = u - (b ? upto[b - 1] : 0);
      g.b = b;
      g.head = static_cast<int>(div64(local, c.head));
      const long long rem = local - g.head * c.head;
      int tl = 0, th = c.tiles - 1; // the last tile whose units begin at or before rem
      while (tl < th) {
        const int mid = (tl + th + 1) >> 1;
        if (c.upto(mid) <= rem)
          tl = mid;
        else
          th = mid - 1;
      }
      const long long cost = c.first + 1ll * tl * c.slope, at = rem - c.upto(tl), to = min(cost, at + (end - u));
      const long long item0 = u - at;
      u += to - at;
      g.row0 = tl * PT_ROWS;
      g.n_rows = min(s.nq * a.G - g.row0, PT_ROWS);
      const int nc = tile_chunks(a, s, g.row0);
      auto chunk_at = [&](long long x) { // chunks that lie before unit x
        return x <= PT_START ? 0 : static_cast<int>(div64((x - PT_START) * nc, cost - PT_START));
      };
      g.chunk0 = chunk_at(at);
      g.chunks = chunk_at(to) - g.chunk0;
      // the first chunk lies with whoever holds the last unit before it is complete
      auto beginner = [&] { return owner(item0 + PT_START + (cost - PT_START + nc - 1) / nc - 1); };
      if (g.chunks == 0) {
        // A request that a short block table cuts off has more units than chunks: a share in its middle can hold
        // none, but the join counts pieces by workers, so it leaves an empty one.
        if (leader && g.chunk0 > 0) {
          a.notes[me].y = beginner();
          const long long pr = 2ll * me * a.rows_per_tile;
#pragma unroll 1
          for (int r = 0; r < g.n_rows; ++r)
            a.part_ml[pr + r] = make_float2(-INFINITY, 0.f);
#pragma unroll 1
          for (int e = 0; e < g.n_rows * a.D; e += 4)
            *reinterpret_cast<float4 *>(a.part_o + pr * a.D + e) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        continue;
      }
      g.slot = -1;
      if (g.chunks < nc) {
        g.slot = 2 * me + (first ? 0 : 1);
        if (leader && g.chunk0 == 0) {
          SplitItem it;
          it.first_slot = g.slot, it.last = owner(item0 + cost - 1);
          it.row0 = g.row0, it.n_rows = g.n_rows, it.q0 = s.q0, it.head = g.head;
          a.items[me] = it, a.notes[me].x = g.n_rows;
        } else if (leader) {
          a.notes[me].y = beginner();
        }
      }
      first = false;
      return true;
    }
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1) attention_paged_tile_kernel(PagedArgs a) {
  using Cfg = PtCfg<D>;
  constexpr int DB = Cfg::DB;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *sQ = smem;                        // [2][Q_BYTES]
  uint8_t *sK = sQ + 2 * Cfg::Q_BYTES;       // [2][K_BYTES]
  uint8_t *sV = sK + 2 * Cfg::K_BYTES;       // [2][K_BYTES]
  uint64_t *bars = reinterpret_cast<uint64_t *>(sV + 2 * Cfg::K_BYTES);
  uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = bars + 6, *v_full = bars + 8,
           *v_empty = bars + 10, *s_full = bars + 12, *p_full = bars + 14, *o_full = bars + 16, *o_free = bars + 18,
           *m_full = bars + 20, *n_full = m_full + PT_SLOTS; // [PT_SLOTS]: scales, NaN flags
  static_assert(20 + 2 * PT_SLOTS <= Cfg::BARS, "barriers");
  float4 *scales = reinterpret_cast<float4 *>(bars + Cfg::BARS); // [PT_SLOTS][8]: K scale, log2 and 1 / V scale
  int4 *v_nan = reinterpret_cast<int4 *>(scales + PT_SLOTS * 8); // [PT_SLOTS][2]: by loader, some value of the tile is NaN
  static_assert(PT_LOADERS <= 8, "one flag each");
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(v_nan + 2 * PT_SLOTS);
  long long *upto = reinterpret_cast<long long *>(smem + Cfg::SMEM + (Cfg::TAIL + 15) / 16 * 16);
  __shared__ long long warp_sum[PT_THREADS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, me = blockIdx.x;
  if (tid == 0)
    a.notes[me] = make_int2(0, -1); // before any way out: the join reads every worker's
  if (smem_u32(smem) & 1023u) { // the swizzled operands need it
    if (tid == 0)
      atomicCAS(a.status, 0, MU_DEV_BAD_LAYOUT);
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // the join waits for the whole grid anyway

  // units of every request, prefix-summed
  long long total;
  {
    const int per = (a.B + PT_THREADS - 1) / PT_THREADS;
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    long long sum = 0;
    for (int b = b0; b < b1; ++b) {
      const Seq s = load_seq(a, b);
      if (s.nq > 0)
        sum += tile_costs(a, s).head * a.Hkv;
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
    long long before = inc - sum;
    total = 0;
#pragma unroll
    for (int w = 0; w < PT_THREADS / 32; ++w) {
      if (w < warp)
        before += warp_sum[w];
      total += warp_sum[w];
    }
    for (int b = b0; b < b1; ++b)
      upto[b] += before;
  }
  if (tid == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 4), mbar_init(&q_empty[x], 1);
      mbar_init(&k_full[x], PT_LOADERS), mbar_init(&k_empty[x], 1);
      mbar_init(&v_full[x], PT_LOADERS), mbar_init(&v_empty[x], 1);
      mbar_init(&s_full[x], 1), mbar_init(&p_full[x], 4);
      mbar_init(&o_full[x], 1), mbar_init(&o_free[x], 4);
    }
    for (int i = 0; i < PT_SLOTS; ++i)
      mbar_init(&m_full[i], 1), mbar_init(&n_full[i], PT_LOADERS);
    for (int i = 0; i < 2 * PT_SLOTS; ++i)
      v_nan[i] = make_int4(0, 0, 0, 0);
    fence_barrier_init();
  }
  __syncthreads();
  if (total == 0)
    return; // nothing allocated yet
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_S = *tmem_slot, tmem_O = tmem_S + 256;

  TileWalk walk(total, me, gridDim.x);
  Segment g{};
  Seq s{};
  // key tiles of the segment that query tile x sees
  auto tiles_of = [&](int x) {
    if (g.n_rows <= x * PT_BQ)
      return 0;
    const int last = g.row0 + min(g.n_rows, (x + 1) * PT_BQ) - 1;
    return min(g.chunks, max(0, (row_limit(a, s, last) + PT_BK - 1) / PT_BK - g.chunk0));
  };
  bool ok = true;
  auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
    if (ok && !mbar_wait(bar, parity)) {
      atomicCAS(a.status, 0, code);
      ok = false;
    }
    return ok;
  };

  if (warp == 0) {
    // ------------------------------ MMA issuer --------------------------------
    if (lane == 0) {
      constexpr uint32_t idesc_qk = make_idesc(0u, 0u, 0u, PT_BQ, PT_BK), idesc_pv = make_idesc(0u, 0u, 1u, PT_BQ, D);
      uint32_t kq = 0, vq = 0, wq[2] = {0, 0}, pt[2] = {0, 0};
      auto issue_qk = [&](int x, int stage) {
        const uint64_t qd = make_smem_desc(smem_u32(sQ + x * Cfg::Q_BYTES), 16, 1024);
        const uint64_t kd = make_smem_desc(smem_u32(sK + stage * Cfg::K_BYTES), 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = static_cast<uint64_t>(((k / 4) * (PT_BQ * 128) + (k % 4) * 32) >> 4);
          umma_f16(tmem_S + x * PT_BK, qd + off, kd + off, idesc_qk, k != 0 ? 1u : 0u);
        }
        umma_commit(&s_full[x]);
      };
      auto issue_pv = [&](int x, int stage, bool accumulate) {
        const uint64_t vd = make_smem_desc(smem_u32(sV + stage * Cfg::K_BYTES), 8192, 1024);
#pragma unroll
        for (int k = 0; k < PT_BK / 16; ++k)
          umma_f16_ts(tmem_O + x * D, tmem_S + x * PT_BK + k * 8,
                      vd + static_cast<uint64_t>(((k / 4) * (DB * 8192) + (k % 4) * 2048) >> 4), idesc_pv,
                      (accumulate || k != 0) ? 1u : 0u);
      };
      while (walk.next(a, upto, g, s, true)) {
        if (!ok) // a wait ran out: other workers' notes still name the items that this one begins
          continue;
        const int nk_x[2] = {tiles_of(0), tiles_of(1)}, nk = max(nk_x[0], nk_x[1]);
        if (nk == 0)
          continue;
        for (int x = 0; x < 2; ++x)
          if (nk_x[x] > 0)
            wait(&q_full[x], wq[x] & 1, MU_DEV_TIMEOUT_MMA);
        if (!wait(&k_full[kq & 1], (kq >> 1) & 1, MU_DEV_TIMEOUT_MMA))
          continue;
        tc_fence_after();
        for (int x = 0; x < 2; ++x)
          if (nk_x[x] > 0) {
            issue_qk(x, kq & 1);
            if (nk_x[x] == 1)
              umma_commit(&q_empty[x]);
          }
        umma_commit(&k_empty[kq & 1]);
        ++kq;
        for (int j = 0; j < nk && ok; ++j) {
          if (!wait(&v_full[vq & 1], (vq >> 1) & 1, MU_DEV_TIMEOUT_MMA))
            break;
          bool k_ready = false;
          for (int x = 0; x < 2 && ok; ++x) {
            if (j >= nk_x[x])
              continue;
            // the first P.V of a work overwrites O_x, which the softmax warps must have read
            wait(&p_full[x], pt[x] & 1, MU_DEV_TIMEOUT_MMA);
            if (j == 0)
              wait(&o_free[x], (wq[x] & 1) ^ 1, MU_DEV_TIMEOUT_MMA);
            if (!ok)
              break;
            ++pt[x];
            tc_fence_after();
            issue_pv(x, vq & 1, j > 0);
            if (j == nk_x[x] - 1)
              umma_commit(&o_full[x]);
            if (j + 1 < nk_x[x]) {
              if (!k_ready) {
                if (!wait(&k_full[kq & 1], (kq >> 1) & 1, MU_DEV_TIMEOUT_MMA))
                  break;
                tc_fence_after();
                k_ready = true;
              }
              issue_qk(x, kq & 1);
              if (j + 1 == nk_x[x] - 1)
                umma_commit(&q_empty[x]);
            }
          }
          if (!ok)
            break;
          umma_commit(&v_empty[vq & 1]);
          ++vq;
          if (j + 1 < nk) {
            umma_commit(&k_empty[kq & 1]);
            ++kq;
          }
        }
        for (int x = 0; x < 2; ++x)
          wq[x] += nk_x[x] > 0;
      }
    }
    __syncwarp();
  } else if (warp <= PT_LOADERS) {
    // ------------------------------ keys and values ---------------------------
    // piece i of a thread: 16 bytes, chunk p % CPK of key p / CPK with p = lt + 224 i
    constexpr int CPK = D / 16, SWEEP = 32 * PT_LOADERS, N = (PT_BK * CPK + SWEEP - 1) / SWEEP;
    const int lt = tid - 32;
    // Three tiles are under way: K and V of tile t are written to shared memory as their stages come free,
    // those of t + 1 are then requested into the same registers, and the pages of t + 2 are looked up. Lane g
    // of every warp keeps group g of 16 keys (one page): where its bytes begin, and how many keys are live.
    struct Tile {
      const int *pages; // the request's row of the block table
      int head, key0, seen;
      bool any;
      int page;       // of group `lane`, as it is in the table
      long long base; // bytes before the group, or -1
    };
    int j = 0, nk = 0;
    auto next_tile = [&](Tile &n) { // and the look-up of its pages
      n.any = true;
      while (j >= nk) {
        if (!walk.next(a, upto, g, s, false)) {
          n.any = false;
          break;
        }
        j = 0, nk = max(tiles_of(0), tiles_of(1));
      }
      n.pages = a.table + 1ll * g.b * a.table_stride;
      n.head = g.head, n.key0 = (g.chunk0 + j) * PT_BK, n.seen = n.any ? s.seen : 0;
      n.page = -1;
      if (lane < 8 && n.key0 + 16 * lane < n.seen)
        n.page = n.pages[a.by_page.div(n.key0 + 16 * lane)];
      ++j;
    };
    auto settle = [&](Tile &n) { // the pages have arrived
      const int key = n.key0 + 16 * lane;
      const bool wanted = lane < 8 && key < n.seen, good = wanted && n.page >= 0 && n.page < a.num_pages;
      if (wanted && !good)
        atomicCAS(a.status, 0, MU_DEV_BAD_PAGE);
      n.base = good ? ((1ll * n.page * a.Hkv + n.head) * a.page_size + a.by_page.mod(key)) * D : -1;
    };
    auto request = [&](const uint8_t *cache, const Tile &n, uint4 (&r)[N]) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int piece = lt + SWEEP * i, key = piece / CPK;
        const long long base = __shfl_sync(~0u, n.base, (key >> 4) & 7);
        const bool live = key < PT_BK && base >= 0 && n.key0 + key < n.seen;
        const uint4 *at = reinterpret_cast<const uint4 *>(cache + (live ? base + (piece & (16 * CPK - 1)) * 16 : 0));
        // zeros first: written after the load they would wait for it, and every load for the one before
        r[i] = make_uint4(0, 0, 0, 0);
        if (live)
          r[i] = __ldg(at);
      }
    };
    auto put = [&](uint8_t *dst, const uint4 &r, int row, int cc) { // 16 elements: two swizzled 16-byte chunks
      *reinterpret_cast<uint4 *>(dst + row * 128 + ((cc ^ (row & 7)) << 4)) =
          make_uint4(f16x2_of_e4m3_lo(r.x), f16x2_of_e4m3_hi(r.x), f16x2_of_e4m3_lo(r.y), f16x2_of_e4m3_hi(r.y));
      *reinterpret_cast<uint4 *>(dst + row * 128 + (((cc + 1) ^ (row & 7)) << 4)) =
          make_uint4(f16x2_of_e4m3_lo(r.z), f16x2_of_e4m3_hi(r.z), f16x2_of_e4m3_lo(r.w), f16x2_of_e4m3_hi(r.w));
    };
    Tile now, soon;
    uint4 kr[N], vr[N];
    float ks = 0.f, vs = 0.f; // this lane's group of the tile `now`
    auto request_scales = [&](const Tile &n) {
      ks = vs = 0.f;
      if (warp == 1 && n.base >= 0) {
        const long long at = 1ll * n.page * a.Hkv + n.head;
        ks = a.ks[at], vs = a.vs[at];
      }
    };
    next_tile(now);
    settle(now);
    if (now.any) {
      request(a.kc, now, kr);
      request(a.vc, now, vr);
      request_scales(now);
      next_tile(soon);
    }
    for (uint32_t t = 0; ok && now.any; ++t) {
      const int slot = t & (PT_SLOTS - 1), stage = t & 1;
      if (warp == 1) { // no page: no weight
        if (lane < 8)
          scales[slot * 8 + lane] = now.base >= 0
                                        ? make_float4(ks, log2f(fmaxf(vs, 0x1p-64f)), 1.f / fmaxf(vs, 0x1p-64f), 0.f)
                                        : make_float4(0.f, -INFINITY, 0.f, 0.f);
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&m_full[slot]);
      }
      settle(soon);
      if (!wait(&k_empty[stage], ((t >> 1) & 1) ^ 1, MU_DEV_TIMEOUT_PRODUCER))
        break;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int piece = lt + SWEEP * i, key = piece / CPK, chunk = piece % CPK;
        if (key < PT_BK)
          put(sK + stage * Cfg::K_BYTES + chunk / 4 * (PT_BK * 128), kr[i], key, chunk % 4 * 2);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&k_full[stage]);
      request(a.kc, soon, kr);
      // NaN values become zeros here; the rows that see them are marked by the softmax warps
      bool nan = false;
#pragma unroll
      for (int i = 0; i < N; ++i)
        nan |= has_nan_e4m3(vr[i].x) | has_nan_e4m3(vr[i].y) | has_nan_e4m3(vr[i].z) | has_nan_e4m3(vr[i].w);
      nan = __any_sync(~0u, nan);
      if (nan) {
        auto clean = [](uint32_t w) {
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            if (((w >> k) & 0x7fu) == 0x7fu)
              w &= ~(0xffu << k);
          return w;
        };
#pragma unroll
        for (int i = 0; i < N; ++i)
          vr[i] = make_uint4(clean(vr[i].x), clean(vr[i].y), clean(vr[i].z), clean(vr[i].w));
      }
      if (lane == 0) {
        reinterpret_cast<int *>(v_nan + 2 * slot)[warp - 1] = nan;
        mbar_arrive(&n_full[slot]);
      }
      __syncwarp();
      if (!wait(&v_empty[stage], ((t >> 1) & 1) ^ 1, MU_DEV_TIMEOUT_PRODUCER))
        break;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int piece = lt + SWEEP * i, key = piece / CPK, chunk = piece % CPK;
        if (key < PT_BK)
          put(sV + stage * Cfg::K_BYTES + ((key >> 6) * DB + chunk / 4) * 8192, vr[i], key & 63, chunk % 4 * 2);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&v_full[stage]);
      request(a.vc, soon, vr);
      request_scales(soon);
      now = soon;
      if (now.any)
        next_tile(soon);
    }
  } else {
    // ---------------- softmax and output: warps 8-11 tile A, warps 12-15 tile B ----------------
    const int x = (warp - 8) >> 2;
    const int q = warp & 3; // tensor-memory lane quarter this warp may access
    const int row = q * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t s_addr = tmem_S + lane_sel + x * PT_BK, o_addr = tmem_O + lane_sel + x * D;
    uint32_t st = 0, wx = 0, t0 = 0; // score tiles and works of this query tile so far; key tiles of the CTA
    while (ok && walk.next(a, upto, g, s, false)) {
      const int nk_all = max(tiles_of(0), tiles_of(1)), nk = tiles_of(x);
      const int my_row = g.row0 + x * PT_BQ + row; // of the request
      const bool live = x * PT_BQ + row < g.n_rows;
      const int limit = live ? row_limit(a, s, my_row) : s.seen + PT_BK; // a row that is not there needs no mask
      const int token = a.by_group.div(my_row), head = g.head * a.G + a.by_group.mod(my_row);
      const uint32_t tile0 = t0;
      t0 += nk_all;
      float m_ref = -INFINITY, l_run = 0.f;
      uint32_t nan_mask[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        nan_mask[i] = 0;
      if (nk > 0) {
        if (!wait(&q_empty[x], (wx & 1) ^ 1, MU_DEV_TIMEOUT_EPILOGUE))
          break;
        // this row of Q, scaled by a power of two to at most 2^15, as fp16. Loops that run once per work are
        // kept short: unrolled, they took longer to fetch as instructions than to execute.
        const __nv_bfloat16 *qp = static_cast<const __nv_bfloat16 *>(a.q) +
                                  (live ? 1ll * (s.q0 + token) * a.q_ld + 1ll * head * D : 0);
        const bool vec = (reinterpret_cast<uintptr_t>(qp) & 15u) == 0;
        auto load8 = [&](int c) { // elements 8c ..
          uint4 u = make_uint4(0, 0, 0, 0);
          if (vec) {
            if (live)
              u = *(reinterpret_cast<const uint4 *>(qp) + c);
          } else if (live) {
            const unsigned short *e = reinterpret_cast<const unsigned short *>(qp) + 8 * c;
            u = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
          }
          return u;
        };
        uint32_t top = 0;
#pragma unroll 1
        for (int c = 0; c < D / 8; c += 8) { // a 128-byte line, its loads together
          uint4 u[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            u[k] = load8(c + k);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(u[k].x & 0x7fff7fffu, u[k].y & 0x7fff7fffu),
                                         __vmaxu2(u[k].z & 0x7fff7fffu, u[k].w & 0x7fff7fffu)));
        }
        top = max(top >> 16, top & 0xffffu) << 16;
        const int e = min(max(static_cast<int>(top >> 23) - 127 - 14, -100), 113);
        const float f = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        const float fac = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * a.scale_log2;
#pragma unroll 1
        for (int c = 0; c < D / 8; c += 2)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint4 u = load8(c + k);
            auto two = [&](uint32_t w) { return f16x2(bf16_lo(w) * f, bf16_hi(w) * f); };
            *reinterpret_cast<uint4 *>(sQ + x * Cfg::Q_BYTES + q_word(row, c + k)) =
                make_uint4(two(u.x), two(u.y), two(u.z), two(u.w));
          }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&q_full[x]);

        for (int j = 0; j < nk && ok; ++j, ++st) {
          const int slot = (tile0 + j) & (PT_SLOTS - 1), lim = limit - (g.chunk0 + j) * PT_BK;
          wait(&s_full[x], st & 1, MU_DEV_TIMEOUT_EPILOGUE);
          // Behind the scores: a query tile that had no part in the key tiles before may be several of the slot's
          // phases ahead, where its parity says nothing; now the scales are there, and those of tile + PT_SLOTS are not.
          if (!wait(&m_full[slot], ((tile0 + j) / PT_SLOTS) & 1, MU_DEV_TIMEOUT_EPILOGUE))
            break;
          tc_fence_after();
          const float4 *sc = scales + slot * 8;
          const bool edge = __any_sync(~0u, lim < PT_BK); // some row of the warp does not see the whole tile
          // 32 columns at a time, the next 32 on their way
          auto sweep = [&](auto &&each) {
            uint32_t r[2][32];
            tmem_ld_32x32(s_addr, r[0]);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              if (h < 3)
                tmem_ld_32x32(s_addr + (h + 1) * 32, r[(h + 1) & 1]);
              each(h, r[h & 1]);
              if (h < 3)
                tmem_ld_wait();
            }
          };
          // pass 1: the row's maximum
          float mx = m_ref;
          auto maxima = [&](auto masked) {
            sweep([&](int h, const uint32_t (&r)[32]) {
#pragma unroll
              for (int gr = 0; gr < 2; ++gr) {
                float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                  float v0 = __uint_as_float(r[gr * 16 + k]), v1 = __uint_as_float(r[gr * 16 + k + 1]);
                  if (decltype(masked)::value) {
                    const int col = h * 32 + gr * 16 + k;
                    v0 = col < lim ? v0 : -INFINITY, v1 = col + 1 < lim ? v1 : -INFINITY;
                  }
                  best[k >> 1 & 1] = max3(best[k >> 1 & 1], v0, v1);
                }
                const float4 c = sc[2 * h + gr];
                const float top = fmaxf(best[0], best[1]);
                if (!decltype(masked)::value || top > -INFINITY) // nothing seen: 0 * inf is no maximum
                  mx = fmaxf(mx, fmaf(top, c.x * fac, c.y));
              }
            });
          };
          if (edge)
            maxima(std::true_type{});
          else
            maxima(std::false_type{});
          if (j == 0) {
            m_ref = mx;
          } else {
            const bool grow = mx > m_ref + 8.f;
            if (__any_sync(~0u, grow)) { // the previous P.V is complete: s_full was committed after it
              const float f2 = grow ? ex2_approx(m_ref - mx) : 1.f;
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld_32x32(o_addr + c * 32, r);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  r[k] = __float_as_uint(__uint_as_float(r[k]) * f2);
                tmem_st_32x32(o_addr + c * 32, r);
              }
              tmem_st_wait();
              l_run *= f2;
              if (grow)
                m_ref = mx;
            }
          }
          const float shift = m_ref == -INFINITY ? 0.f : PT_W_EXP - m_ref;
          // pass 2: weights, back over scores already read
          auto weights = [&](auto masked) {
            sweep([&](int h, const uint32_t (&r)[32]) {
              uint32_t pk[16];
#pragma unroll
              for (int gr = 0; gr < 2; ++gr) {
                const float4 c = sc[2 * h + gr];
                const float mul = c.x * fac, add = c.y + shift;
                const uint64_t mul2 = f32x2_pack(mul, mul), add2 = f32x2_pack(add, add);
                uint64_t sum2 = f32x2_pack(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                  float y0, y1;
                  f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(r[gr * 16 + k]), __uint_as_float(r[gr * 16 + k + 1])),
                                         mul2, add2), y0, y1);
                  if (decltype(masked)::value) {
                    const int col = h * 32 + gr * 16 + k;
                    y0 = col < lim ? y0 : -INFINITY, y1 = col + 1 < lim ? y1 : -INFINITY;
                  }
                  y0 = ex2_approx(y0), y1 = ex2_approx(y1);
                  sum2 = f32x2_add(sum2, f32x2_pack(y0, y1));
                  pk[gr * 8 + k / 2] = f16x2(y0, y1);
                }
                float s0, s1;
                f32x2_unpack(sum2, s0, s1);
                l_run = fmaf(s0 + s1, c.z, l_run);
              }
              tmem_st_32x16(s_addr + h * 16, pk); // columns below 16 (h + 1): read, or in registers
            });
          };
          if (edge)
            weights(std::true_type{});
          else
            weights(std::false_type{});
          if (!wait(&n_full[slot], ((tile0 + j) / PT_SLOTS) & 1, MU_DEV_TIMEOUT_EPILOGUE))
            break;
          const int4 some = v_nan[2 * slot], more = v_nan[2 * slot + 1];
          if (some.x | some.y | some.z | some.w | more.x | more.y | more.z) { // which dimensions of the keys this row sees are NaN
            const int key0 = (g.chunk0 + j) * PT_BK, see = min(min(PT_BK, lim), s.seen - key0);
            for (int k = 0; k < see; ++k) {
              const int page = a.table[1ll * g.b * a.table_stride + a.by_page.div(key0 + k)];
              if (page < 0 || page >= a.num_pages)
                continue;
              const uint32_t *v = reinterpret_cast<const uint32_t *>(
                  a.vc + ((1ll * page * a.Hkv + g.head) * a.page_size + a.by_page.mod(key0 + k)) * D);
#pragma unroll
              for (int w = 0; w < D / 4; ++w) {
                const uint32_t u = v[w];
#pragma unroll
                for (int b = 0; b < 4; ++b)
                  if (((u >> (8 * b)) & 0x7fu) == 0x7fu)
                    nan_mask[w >> 3] |= 1u << ((w & 7) * 4 + b);
              }
            }
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0)
            mbar_arrive(&p_full[x]);
        }
        if (!wait(&o_full[x], wx & 1, MU_DEV_TIMEOUT_EPILOGUE))
          break;
        tc_fence_after();
      }
      // ---- output: rows of bfloat16, or a piece for the join. Through this warp's rows of Q's tile (every
      // product that reads them is done), so that rows leave 16 lanes at a time: 16-byte stores a row apart
      // wait on each other's latency.
      const float inv = g.slot >= 0 ? 1.f : l_run == 0.f ? 0.f : 1.f / l_run;
      const long long pr = 1ll * max(g.slot, 0) * a.rows_per_tile + x * PT_BQ + row;
      constexpr int PER_ROW = D / 8; // 16-byte words
      auto cell = [&](int r, int c) { return reinterpret_cast<uint4 *>(sQ + x * Cfg::Q_BYTES + q_word(q * 32 + r, c)); };
      const long long my_out = live ? 1ll * (s.q0 + token) * a.out_ld + 1ll * head * D : -1;
      auto rows_out = [&](auto &&to) { // the staged rows, coalesced: to(row of the warp, word) takes 16 bytes
        __syncwarp();
#pragma unroll 2
        for (int i = 0; i < PER_ROW; ++i) {
          const int r = i * (32 / PER_ROW) + lane / PER_ROW, c = lane % PER_ROW;
          to(r, c, *cell(r, c));
        }
        __syncwarp();
      };
      const bool piece = g.slot >= 0;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (nk > 0) {
          tmem_ld_32x32(o_addr + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            r[k] = 0;
        }
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
          nan = c == i ? nan_mask[i] : nan;
        if (__any_sync(~0u, nan != 0))
#pragma unroll
          for (int k = 0; k < 32; ++k)
            r[k] = nan >> k & 1u ? 0x7fffffffu : r[k];
        if (piece) { // a half of the dimensions as floats fills the row
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            *cell(lane, c % (D / 64) * 8 + k / 4) = make_uint4(r[k], r[k + 1], r[k + 2], r[k + 3]);
          if (c % (D / 64) == D / 64 - 1)
            rows_out([&](int w, int word, const uint4 &v) {
              if (x * PT_BQ + q * 32 + w < g.n_rows)
                *reinterpret_cast<uint4 *>(a.part_o + (pr - lane + w) * D + c / (D / 64) * (D / 2) + word * 4) = v;
            });
        } else {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            auto two = [&](int i) {
              return pack_bf16x2(__uint_as_float(r[k + i]) * inv, __uint_as_float(r[k + i + 1]) * inv);
            };
            *cell(lane, c * 4 + k / 8) = make_uint4(two(0), two(2), two(4), two(6));
          }
        }
      }
      if (!piece)
        rows_out([&](int w, int word, const uint4 &v) {
          const long long off = __shfl_sync(~0u, my_out, w);
          if (off < 0)
            return;
          __nv_bfloat16 *op = static_cast<__nv_bfloat16 *>(a.out) + off + 8 * word;
          if ((reinterpret_cast<uintptr_t>(op) & 15u) == 0) {
            *reinterpret_cast<uint4 *>(op) = v;
          } else {
            unsigned short *e = reinterpret_cast<unsigned short *>(op);
            const uint32_t half[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; ++k)
              e[k] = static_cast<unsigned short>(half[k >> 1] >> (16 * (k & 1)));
          }
        });
      if (live && g.slot >= 0)
        a.part_ml[pr] = make_float2(m_ref == -INFINITY ? -INFINITY : m_ref - PT_W_EXP, l_run);
      if (nk > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&o_free[x]); // O_x may be overwritten by the next work
        ++wx;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0)
    tmem_dealloc(tmem_S, 512);
}

// 0 ok, 2 CUDA error. D is 64 or 128; one worker per SM.
template <int D> static int launch_tile_d(const PagedArgs &a, int num_sms, cudaStream_t st) {
  constexpr size_t fixed = PtCfg<D>::SMEM + (PtCfg<D>::TAIL + 15) / 16 * 16;
  static PerDeviceOnce once;
  if (once.get() < 0) {
    if (cudaFuncSetAttribute(attention_paged_tile_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(fixed + 8 * MU_PAGED_TILE_MAX_REQUESTS)) != cudaSuccess)
      return 2;
    once.set(1);
  }
  attention_paged_tile_kernel<D><<<num_sms, PT_THREADS, fixed + 8ull * a.B, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 2;
}
int launch_attention_paged_tile(const PagedArgs &a, int num_sms, cudaStream_t st) {
  return a.D == 128 ? launch_tile_d<128>(a, num_sms, st) : launch_tile_d<64>(a, num_sms, st);
}

} // namespace mu
