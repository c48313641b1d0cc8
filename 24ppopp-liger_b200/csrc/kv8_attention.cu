// Attention over the paged 8-bit cache for few query rows per key head (a decode step, a few drafted tokens).
//
// Bound by HBM: every code of the cache is read once and used for all query rows of its key head.  What has to be done per code
// is kept small enough to hide under that: a code becomes an fp16 number (exactly) with one or two instructions and goes
// into mma.sync, 16 keys x 8 query rows at a time.
//
//   S^T[key, row] = K Q^T    A = 16 keys x 16 dims, B = 16 dims x 8 rows.  Which dims stand at which k of a product does not
//                            matter as long as A and B agree, so a lane takes 16 contiguous bytes of a key at a time.
//   O^T[dim, row] += V^T P^T A = 16 dims x 16 keys: a lane holds 16 contiguous dims of four keys and pairs the keys' bytes.
//                            P^T comes out of the S^T accumulators by an 8x8 transpose (movmatrix).
//
// Rows are (new token, head of the group) pairs, 4, 8, 16 or 24 of them a tile.  Scales: S is multiplied by its key block's scale in
// fp32.  The value scale goes into P: w = p * (scale / reference), where the reference follows the scales (the accumulators are rescaled
// when it moves), so that w stays where fp16 is precise.  P is split into a leading and a
// trailing fp16 part, two products, so that its rounding does not show in the result.  With at most 4 rows both parts go into one product: columns 4 .. 7
// are the rows again, with the trailing parts.  (The GPU runs into its power limit here, 1000 W, and the products are what can be saved:
// 32 x 2049 tokens of 96 heads, e4m3, over seconds 286 us with two products, 271 us with one, 250 us for the copies alone.)  The reference
// score follows the steps' largest scores up and down, but only where one leaves it (kAbove, kBelow), which a warp finds with one vote, and
// a reduction where a lane has no score near it: so a step's weights do not fall out of fp16's range because another step's were larger (2 .. 3 % of
// the calls below).  fp16 ends at 2^-24: a weight is off by at most 2^-22 of itself or 2^-21 of the step's largest weight and value scale (where the
// reference score is as low as it goes: 2^-74 of the row's sum so far), whichever is more.
//
// Work is counted in places: a tile (sequence, key head, row tile) has one for each step of 16 keys and kTileCost for what
// it costs to begin one.  All tiles' places form one line, and every warp takes an equal share of it, whatever the lengths
// are; warps do not wait for one another before the end.  Where a share begins or ends inside a tile the partial (maximum, sum,
// accumulator) goes to scratch and a second, small kernel joins the parts; parts of one tile that neighbouring warps of a CTA have are
// joined in shared memory first (48 x up to 16384 tokens of 8 heads: 71 -> 65 us).  Short calls with few
// tiles give each tile to the eight warps of a CTA instead, which join in shared memory.  Either way a warp fills a ring of
// stages of its own with 16-byte asynchronous copies.
//
// Measured (device time in a row of calls): 32 x 2049 tokens, 96 heads of 128, e4m3: 257 us, 6.3 TB/s (96 % of the copy rate; 277 us over
// seconds); 48 x up to 16384 tokens, 8 heads of 128 for 64 queries, int8: 67 .. 73 us, 4.4 .. 4.8 TB/s; 2 x 150001 tokens, 4 heads of 128
// for 20 queries, e4m3: 58 .. 62 us, 5.0 .. 5.3 TB/s.  What the shorter calls miss is some 7 us until the first codes arrive (lengths, table,
// codes: one after the other) and some 5 us for the join.  5 drafted tokens of 12 sequences behind up to 6000, 8 heads for 32 queries, int8:
// 45 us, 2.0 TB/s; here the work between the copies is what takes time (29 us without it): 72 products a step of 16 keys, with two warps
// on a scheduler since 24 rows fill the registers.
#include <cfloat>

#include "kv8_attention.cuh"

namespace liger {
namespace {

constexpr int kWarps = 4;            // of a CTA whose warps have shares of their own
constexpr int kWholeWarps = 8;       // of a CTA that has a whole tile
constexpr int kStep = 16;            // keys of a step
constexpr int kTileCost = 4;         // what it costs to begin a tile, in steps
constexpr int kMinPlaces = 8;        // places that are worth a warp
// Rows a key head up to which this kernel is taken.  A tile has 24 at most, and the cache is read once for each.  12 x 4000 tokens, 8
// heads, int8, here and in kv8_attention_tc_kernel: 24 rows of 128 50 and 82 us, 48 rows 83 and 86 (of 64: 63 and 77), 56 rows 114 and 87 (84
// and 77); e4m3: 48 rows 78 and 84, 56 rows 107 and 86.
constexpr int kFewRows = 48;
constexpr float kLog2e = 1.4426950408889634f;
// Where the weights lie among fp16 numbers (in log2 units): the reference score has weight 2^10, a score up to 4 above it and a value scale up to
// twice the reference come on top.  A step's largest score is at most 12 below the reference score, unless a reference that low would make the row's
// sum so far more than 2^50.
constexpr float kUnit = 10.0f, kAbove = 4.0f, kBelow = 12.0f, kMostSum = 50.0f;

// ROWS: of a tile, 4, 8, 16 or 24
template <int D, int ROWS, int WHOLE>
struct Cfg {
  static constexpr int NT = (ROWS + 7) / 8;                          // groups of 8 columns of a product
  static constexpr int kWarps = WHOLE ? kWholeWarps : liger::kWarps;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kCtas = WHOLE ? 1 : NT == 1 ? 3 : 2;          // resident per SM
  static constexpr int kStage = 2 * kStep * D;                       // K and V of a step
  static constexpr int kStages = (NT == 1 || WHOLE ? 4 : 6) * (128 / D);
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kMerge = kWarps * ROWS * (D + 4) * 4;         // accumulators of a CTA's warps, in the place of the rings
  static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
  static constexpr int kPart = ROWS * (D + 2);                       // floats of a partial result: maxima, sums, accumulators
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// an entry without keys still has rows to fill with zeros
__device__ __forceinline__ int steps_of(const Entry& e) { return max(1, (e.len + kStep - 1) / kStep); }
__device__ __forceinline__ int places_of(const Entry& e) { return steps_of(e) + kTileCost; }
template <int ROWS>
__device__ __forceinline__ long long line_of(const Kv8AttnParams& p, const Entry& e) {
  return (long long)p.c.kv_heads * row_tiles<ROWS>(p, e) * places_of(e);
}

// 16-byte chunk `c` of key `r` of a step.  The xor spreads both ways of reading over all banks: a lane quad reads a key
// across (K), and eight lanes with one dim range each read four keys (V).
template <int D>
__device__ __forceinline__ int stage_at(int r, int c) {
  if (D == 128) return r * 128 + ((c ^ ((r & 6) ^ ((r & 1) << 2))) << 4);
  return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (r & 6)) << 4);  // two keys a line
}

template <int D, int TYPE, int ROWS, int WHOLE>
__global__ void __launch_bounds__(Cfg<D, ROWS, WHOLE>::kThreads, Cfg<D, ROWS, WHOLE>::kCtas) kv8_attention_kernel(const Kv8AttnParams p) {
  using C = Cfg<D, ROWS, WHOLE>;
  constexpr int NT = C::NT;
  constexpr bool kPacked = ROWS == 4;             // columns 4 .. 7 are rows 0 .. 3 again, with the trailing parts of the weights
  constexpr int kCols = kPacked ? 4 : 8;          // rows of a group of columns
  constexpr int kWarps = C::kWarps, kThreads = C::kThreads;
  constexpr int kKk = D / 16;                     // k-steps of a score product = dim tiles of an output product
  constexpr int kStride = WHOLE ? kWarps : 1;     // the warps of a whole tile take every eighth step
  extern __shared__ __align__(128) uint8_t smem_kv8[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem_kv8 + warp * C::kStages * C::kStage;
  const uint32_t ring_u = smem_u32(ring);
  wait_for_stream();

  // the places [at, end) of the line, beginning in entry b whose places start at b_first
  long long at = 0, end = 0, b_first = 0;
  int b;
  Kv8Deal deal{};
  const int worker = blockIdx.x * kWarps + warp;
  Entry e;
  bool grouped = false;
  __shared__ int s_follows[kWarps], s_rows[kWarps];
  __shared__ float* s_part[kWarps];
  if constexpr (WHOLE) {
    b = blockIdx.y;
    e = load_entry(p, b, blockIdx.x == 0 && threadIdx.x == 0);
    if ((int)blockIdx.x >= p.c.kv_heads * row_tiles<ROWS>(p, e)) return;
    at = (long long)blockIdx.x * places_of(e);
    end = at + places_of(e);
  } else {
    __shared__ Kv8Shares<kWarps> shares;
    if (lane == 0) s_follows[warp] = s_rows[warp] = 0;
    find_shares<kThreads>(p, kMinPlaces, [&](const Entry& x) { return line_of<ROWS>(p, x); }, shares);
    deal = shares.deal;
    b = shares.b[warp];
    b_first = shares.first[warp];
    if (!p.by_tile && lane == 0) p.records[worker].first = -1;
    if (b >= 0) {
      at = deal.begin(worker);
      end = deal.begin(worker + 1);
      e = load_entry(p, b, false);
    }
  }
  const long long share0 = at;

  while (at < end) {
    const int steps = steps_of(e), places = places_of(e);
    int place;
    const int tile = (int)divide(at - b_first, places, place);
    const int left = (int)((long long)(places - place) < end - at ? places - place : end - at);  // places of the share in this tile
    const int tiles = row_tiles<ROWS>(p, e);
    const int head = min(tile / tiles, p.c.kv_heads - 1), row_base = (tile % tiles) * ROWS;
    // a share that ends before a tile's first step leaves the tile to the next
    const int s_begin = max(0, place - kTileCost), s_end = max(0, place + left - kTileCost);
    const int rows = e.n * p.group;
    const bool complete = s_begin == 0 && s_end == steps;
    // Parts of one tile that neighbouring warps have are joined here: a warp whose share is a tile's inside follows the warp before
    const long long tile_end = b_first + (long long)(tile + 1) * places;
    const bool follows = !WHOLE && warp > 0 && at == share0 && s_begin > 0 && end < tile_end;
    const bool leads = !WHOLE && s_end > 0 && warp + 1 < kWarps && worker + 1 < deal.used && deal.begin(worker + 2) < tile_end;
   if (s_end > 0) {
    if (!WHOLE && lane == 0 && s_begin == 0)  // who begins a tile knows who ends it
      leave_record(p, worker, complete, complete ? 0 : deal.worker_of(tile_end - 1), e, b, tile, head, row_base);
    // this lane's rows: as B operand row g of each n-tile, as accumulator column 2t, 2t + 1
    uint32_t qf[NT][kKk][2];
    int limit[NT][2], limit_min = e.len;
    uint32_t idle = 0;  // columns without a row, bit by bit
    auto load_rows = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = row_base + nt * 8 + g % kCols;
        uint4 x[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) x[i] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
          const int token = r / p.group;
          const __half* src = p.q + (p.e.q_offsets ? (long long)(e.row0 + token) * p.q_token_stride
                                                   : (long long)b * p.q_batch_stride + (long long)token * p.q_token_stride) +
                              (long long)(head * p.group + r % p.group) * p.q_head_stride;
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            x[2 * h] = kv8_ld(reinterpret_cast<const uint4*>(src + h * 64 + t * 16));
            x[2 * h + 1] = kv8_ld(reinterpret_cast<const uint4*>(src + h * 64 + t * 16 + 8));
          }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          qf[nt][2 * i][0] = x[i].x; qf[nt][2 * i][1] = x[i].y;
          qf[nt][2 * i + 1][0] = x[i].z; qf[nt][2 * i + 1][1] = x[i].w;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int rc = row_base + nt * 8 + (2 * t + c) % kCols;
          if (rc >= rows) idle |= 1u << (nt * 8 + 2 * t + c);
          limit[nt][c] = rc >= rows ? 0 : p.causal ? min(e.len, max(0, e.len - e.n + rc / p.group + 1)) : e.len;
        }
      }
      if (p.causal) limit_min = min(e.len, max(0, e.len - e.n + row_base / p.group + 1));
    };
    if (NT > 2) load_rows();  // while the first steps are under way, where there are registers for both

    // this warp's steps: s_first + i * kStride, i < count (an entry without keys has none)
    const int s_first = s_begin + (WHOLE ? warp : 0);
    const int count = e.len > 0 && s_first < s_end ? (s_end - s_first + kStride - 1) / kStride : 0;
    const int* row_table = p.c.table + (size_t)e.slot * p.c.max_pages;
    const int page_mask = (1 << p.c.page_shift) - 1;
    // page and scales of 32 steps, one per lane: `now` for steps being copied, the lookups of the next 32 under way
    auto lookup = [&](int i0, int& page, float& ks, float& vs) {
      const int i = i0 + lane;
      page = -1;
      ks = vs = 0.0f;
      if (i < count) {
        const int key = (s_first + i * kStride) * kStep;
        page = kv8_ld(row_table + (key >> p.c.page_shift));
        if (page < 0 || page >= p.c.num_pages) {
          report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAttention + 2, b, (unsigned)page);
          page = -1;
        } else {
          const size_t ph = (size_t)page * p.c.kv_heads + head;
          const size_t blk = (ph << (p.c.page_shift - p.c.block_shift)) + ((key & page_mask) >> p.c.block_shift);
          ks = kv8_ld(p.c.ks + blk);
          vs = kv8_ld(p.c.vs + blk);
          if (!(ks >= 0.0f && ks < INFINITY)) ks = NAN;
          if (!(vs >= 0.0f && vs < INFINITY)) vs = NAN;
        }
      }
    };
    int page_even, page_odd;  // of windows of 32 steps, by the window's parity: the one in use and the next
    float ks_even, ks_odd, vs_even, vs_odd;
    lookup(0, page_even, ks_even, vs_even);
    lookup(32, page_odd, ks_odd, vs_odd);

    auto copy_step = [&](int i) {
      if (i < count) {
        const int page = __shfl_sync(0xffffffffu, (i >> 5) & 1 ? page_odd : page_even, i & 31);
        if (page >= 0) {
          const int key = (s_first + i * kStride) * kStep;
          const size_t src = ((((size_t)page * p.c.kv_heads + head) << p.c.page_shift) + (key & page_mask)) * D;
          const uint32_t dst = ring_u + (i % C::kStages) * C::kStage;
          constexpr int kChunks = D / 16;
#pragma unroll
          for (int j = 0; j < kStep * D / 512; ++j) {
            const int r = lane / kChunks + j * (32 / kChunks), c = lane % kChunks;
            const int off = stage_at<D>(r, c);
            cp_async16(dst + off, p.c.k + src + r * D + c * 16);
            cp_async16(dst + kStep * D + off, p.c.v + src + r * D + c * 16);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < C::kStages - 1; ++i) copy_step(i);

    if (NT <= 2) load_rows();
    float m_ref[NT][2], l_run[NT][2], v_ref = 0.0f, v_back = 0.0f, v_top = 0.0f;  // m_ref: a reference score less kUnit
    float o[NT][kKk][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_ref[nt][0] = m_ref[nt][1] = -INFINITY;
      l_run[nt][0] = l_run[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < kKk; ++i) { o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f; }
    }

#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      // window boundary: steps up to i + kStages - 2 are under way; once the copies reach window w + 1, window w - 1 is done with
      if ((i & 31) == 0 && i > 0) {
        if ((i >> 5) & 1) lookup(i + 32, page_even, ks_even, vs_even);
        else lookup(i + 32, page_odd, ks_odd, vs_odd);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
      __syncwarp();
      const int odd = (i >> 5) & 1;
      const int page = __shfl_sync(0xffffffffu, odd ? page_odd : page_even, i & 31);
      const float ks = __shfl_sync(0xffffffffu, odd ? ks_odd : ks_even, i & 31);
      const float vs = __shfl_sync(0xffffffffu, odd ? vs_odd : vs_even, i & 31);
      const int key0 = (s_first + i * kStride) * kStep;
      const uint8_t* sk = ring + (i % C::kStages) * C::kStage;
      uint8_t* sv = ring + (i % C::kStages) * C::kStage + kStep * D;
      if (page >= 0) {
        if (key0 + kStep > e.len) {  // behind the last key lies anything: it must not meet a weight of 0 as a NaN
          constexpr int kChunks = D / 16;
          for (int j = lane; j < kStep * kChunks; j += 32)
            if (key0 + j / kChunks >= e.len) *reinterpret_cast<uint4*>(sv + stage_at<D>(j / kChunks, j % kChunks)) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
        const bool masked = key0 + kStep > limit_min;
        // S^T = K Q^T
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          const uint4 ka = *reinterpret_cast<const uint4*>(sk + stage_at<D>(g, t + 4 * h));
          const uint4 kb = *reinterpret_cast<const uint4*>(sk + stage_at<D>(g + 8, t + 4 * h));
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a = kv8_bias<TYPE>(wa[w]), c = kv8_bias<TYPE>(wb[w]);
            const uint32_t a0 = kv8_pair<TYPE, 0>(a), a2 = kv8_pair<TYPE, 1>(a), a1 = kv8_pair<TYPE, 0>(c), a3 = kv8_pair<TYPE, 1>(c);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a0, a1, a2, a3, qf[nt][4 * h + w][0], qf[nt][4 * h + w][1]);
          }
        }
        // scores in units of log2; s[.][0], [1]: key g, rows 2t, 2t + 1; s[.][2], [3]: key g + 8
        const float xs = ks * p.scale_log2;
        float top = -INFINITY, low = INFINITY;  // of the lane's columns, each by its two keys; a column without a reference or a score is no number and drops out
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 4; ++c) s[nt][c] *= xs;
          if (masked) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (key0 + g + (c >> 1) * 8 >= limit[nt][c & 1]) s[nt][c] = -INFINITY;
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float above = fmaxf(s[nt][c], s[nt][c + 2]) - m_ref[nt][c];
            top = fmaxf(top, above);
            low = fminf(low, above);
          }
        }
        // Some score is too far above its reference, or a lane has none near it; in the second case a column may still have one in another lane.
        bool leaves = __any_sync(0xffffffffu, top > kUnit + kAbove || low < kUnit - kBelow);
        if (leaves) {
          uint32_t near = top > kUnit + kAbove ? 1u << 31 : idle;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (fmaxf(s[nt][c], s[nt][c + 2]) - m_ref[nt][c] >= kUnit - kBelow) near |= 1u << (nt * 8 + 2 * t + c);
          leaves = __reduce_or_sync(0xffffffffu, near) != (1u << (NT * 8)) - 1u;
        }
        if (leaves) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(s[nt][c], s[nt][c + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              float sum = l_run[nt][c];
              sum += __shfl_xor_sync(0xffffffffu, sum, 4);
              sum += __shfl_xor_sync(0xffffffffu, sum, 8);
              sum += __shfl_xor_sync(0xffffffffu, sum, 16);
              if (mx > m_ref[nt][c] + (kUnit + kAbove) || (mx < m_ref[nt][c] + (kUnit - kBelow) && mx > -INFINITY)) {
                const float to = fmaxf(mx - kUnit, m_ref[nt][c] - (kMostSum - __log2f(sum)));
                const float alpha = exp2_approx(m_ref[nt][c] - to);  // 0 the first time
                m_ref[nt][c] = to;
                l_run[nt][c] *= alpha;
#pragma unroll
                for (int d = 0; d < kKk; ++d) { o[nt][d][c] *= alpha; o[nt][d][c + 2] *= alpha; }
              }
            }
          }
        }
        // weights.  The value scale relative to the reference, which moves where a scale leaves it (twice, a quarter)
        float rel = vs * v_back;
        if (!(rel <= 2.0f && rel >= 0.25f) && vs > fmaxf(v_top * kScaleVanishes, FLT_MIN)) {
          const float back = v_ref / vs;  // 0 the first time
          v_ref = vs;
          v_top = fmaxf(v_top, vs);
          v_back = 1.0f / vs;
          rel = 1.0f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < kKk; ++d) { o[nt][d][0] *= back; o[nt][d][1] *= back; o[nt][d][2] *= back; o[nt][d][3] *= back; }
        }
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float m = m_ref[nt][c & 1];
            const float pr = exp2_approx(s[nt][c] - (m == -INFINITY ? 0.0f : m));
            l_run[nt][c & 1] += pr;
            w[c] = pr * rel;
          }
          if (masked) {  // a key that is not seen has no weight, whatever its scale is
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (s[nt][c] == -INFINITY) w[c] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const __half2 hi = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
            const float2 back = __half22float2(hi);
            const uint32_t lead = *reinterpret_cast<const uint32_t*>(&hi), trail = pack_half2(w[2 * i] - back.x, w[2 * i + 1] - back.y);
            ph[nt][i] = transpose8x8(kPacked && t >= 2 ? trail : lead);
            if (!kPacked) pl[nt][i] = transpose8x8(trail);
          }
        }
        // O^T += V^T P^T
        constexpr int kWords = D / 32;  // 4-byte words of dims that a lane holds of each key
        uint32_t vw[4][kWords];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = 2 * t + (j & 1) + (j >> 1) * 8;
          if (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(sv + stage_at<D>(key, g));
            vw[j][0] = x.x; vw[j][1] = x.y; vw[j][2 % kWords] = x.z; vw[j][3 % kWords] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sv + stage_at<D>(key, g >> 1) + (g & 1) * 8);
            vw[j][0] = x.x; vw[j][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          const uint32_t x0 = kv8_bias<TYPE>(vw[0][w]), x1 = kv8_bias<TYPE>(vw[1][w]), x2 = kv8_bias<TYPE>(vw[2][w]), x3 = kv8_bias<TYPE>(vw[3][w]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t ab = __byte_perm(x0, x1, half ? 0x7362 : 0x5140), cd = __byte_perm(x2, x3, half ? 0x7362 : 0x5140);
            const uint32_t a0 = kv8_pair<TYPE, 0>(ab), a1 = kv8_pair<TYPE, 1>(ab), a2 = kv8_pair<TYPE, 0>(cd), a3 = kv8_pair<TYPE, 1>(cd);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[nt][2 * w + half], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
              if (!kPacked) mma_f16(o[nt][2 * w + half], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
            }
          }
        }
      }
      __syncwarp();  // all lanes have read stage i before it is filled again
      copy_step(i + C::kStages - 1);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // this warp's sums over the keys' lanes
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], 4);
        l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], 8);
        l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], 16);
        if (kPacked) {  // both parts of the weights
#pragma unroll
          for (int d = 0; d < kKk; ++d) {
            o[nt][d][c] += __shfl_xor_sync(0xffffffffu, o[nt][d][c], 2);
            o[nt][d][c + 2] += __shfl_xor_sync(0xffffffffu, o[nt][d][c + 2], 2);
          }
        }
      }
    if (WHOLE) {
      __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
      float* merge = reinterpret_cast<float*>(smem_kv8);
      __syncthreads();  // the rings are done with
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = nt * 8 + 2 * t + c;
          if (kPacked && t >= 2) continue;
          if (g == 0) { s_m[warp][r] = m_ref[nt][c]; s_l[warp][r] = l_run[nt][c]; }
          float* dst = merge + (warp * ROWS + r) * (D + 4) + g * (D / 8);
#pragma unroll
          for (int d = 0; d < kKk; d += 2)
            *reinterpret_cast<float4*>(dst + 2 * d) = make_float4(o[nt][d][c] * v_ref, o[nt][d][c + 2] * v_ref, o[nt][d + 1][c] * v_ref, o[nt][d + 1][c + 2] * v_ref);
        }
      __syncthreads();
      for (int i = threadIdx.x; i < ROWS * D / 4; i += kThreads) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        if (row_base + r >= rows) break;
        float m = s_m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w][r]);
        float l = 0.0f;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float lw = s_l[w][r];
          const float f = lw == 0.0f ? 0.0f : lw == lw ? exp2_approx(s_m[w][r] - m) : 1.0f;  // saw nothing / a NaN stays
          const float4 x = *reinterpret_cast<const float4*>(merge + (w * ROWS + r) * (D + 4) + d);
          l += f * lw;
          a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
        }
        const int token = (row_base + r) / p.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        __half* dst = p.out + (size_t)(e.row0 + token) * p.ldo + (size_t)(head * p.group + (row_base + r) % p.group) * D + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(a.x * inv, a.y * inv), pack_half2(a.z * inv, a.w * inv));
      }
      return;
    }
    float* part = p.parts + (size_t)(2 * worker + (at == share0 && s_begin > 0 ? 0 : 1)) * C::kPart;
    grouped = follows || leads;
    if (grouped) {  // in the place of this warp's ring
      if (lane == 0) {
        s_follows[warp] = follows;
        s_rows[warp] = min(ROWS, rows - row_base);
        s_part[warp] = part;
      }
      part = reinterpret_cast<float*>(ring);
      __syncwarp();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * t + c;
        if (r >= ROWS || row_base + r >= rows) continue;
        if (complete) {
          const int token = (row_base + r) / p.group;
          const float inv = l_run[nt][c] == 0.0f ? 0.0f : v_ref / l_run[nt][c];
          __half* dst = p.out + (size_t)(e.row0 + token) * p.ldo + (size_t)(head * p.group + (row_base + r) % p.group) * D + g * (D / 8);
#pragma unroll
          for (int d = 0; d < kKk; d += 4)
            *reinterpret_cast<uint4*>(dst + 2 * d) = make_uint4(pack_half2(o[nt][d][c] * inv, o[nt][d][c + 2] * inv),
                                                                pack_half2(o[nt][d + 1][c] * inv, o[nt][d + 1][c + 2] * inv),
                                                                pack_half2(o[nt][d + 2][c] * inv, o[nt][d + 2][c + 2] * inv),
                                                                pack_half2(o[nt][d + 3][c] * inv, o[nt][d + 3][c + 2] * inv));
        } else {
          if (g == 0) { part[r] = m_ref[nt][c]; part[ROWS + r] = l_run[nt][c]; }
          float* dst = part + 2 * ROWS + r * D + g * (D / 8);
#pragma unroll
          for (int d = 0; d < kKk; d += 2)
            *reinterpret_cast<float4*>(dst + 2 * d) = make_float4(o[nt][d][c] * v_ref, o[nt][d][c + 2] * v_ref, o[nt][d + 1][c] * v_ref, o[nt][d + 1][c + 2] * v_ref);
        }
      }
   }

    at += left;
    if (at < end && at == b_first + (long long)p.c.kv_heads * tiles * places) {
      b_first = at;
      do {
        if (++b >= p.e.batch) {  // only if the lengths changed under the call
          e.n = 0;
          end = at;
          break;
        }
        e = load_entry(p, b, false);
      } while (e.n == 0);  // entries without new tokens have no place in the line
    }
  }
  if (WHOLE) return;

  // the parts of tiles that neighbouring warps share
  __syncthreads();
  if (!grouped) return;
  int lead = warp, last = warp;
  while (s_follows[lead]) --lead;
  while (last + 1 < kWarps && s_follows[last + 1]) ++last;
  const float* parts = reinterpret_cast<const float*>(smem_kv8);
  constexpr int kRingFloats = C::kStages * C::kStage / 4;
  float* part = s_part[lead];
  for (int i = (warp - lead) * 32 + lane; i < s_rows[lead] * (D / 4); i += (last - lead + 1) * 32) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    for (int w = lead; w <= last; ++w) m = fmaxf(m, parts[w * kRingFloats + r]);
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = lead; w <= last; ++w) {
      const float* q = parts + w * kRingFloats;
      const float lw = q[ROWS + r];
      const float f = lw == 0.0f ? 0.0f : lw == lw ? exp2_approx(q[r] - m) : 1.0f;  // saw nothing / a NaN stays
      const float4 x = *reinterpret_cast<const float4*>(q + 2 * ROWS + r * D + d);
      l = fmaf(f, lw, l);
      a.x = fmaf(f, x.x, a.x); a.y = fmaf(f, x.y, a.y); a.z = fmaf(f, x.z, a.z); a.w = fmaf(f, x.w, a.w);
    }
    if (d == 0) { part[r] = m; part[ROWS + r] = l; }
    *reinterpret_cast<float4*>(part + 2 * ROWS + r * D + d) = a;
  }
}

Kv8AttnPlan plan_of(const liger_kv8_cache* c, const liger_kv8_attention_args* a, int sm_count) {
  Kv8AttnPlan p;
  const long long rows = (long long)a->q_len * (a->heads / c->kv_heads);
  const bool tc = rows > kFewRows && a->scale > 0.0f;
  p.rows = tc ? kTcRows : rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 24;
  p.live = (int)(rows < p.rows ? rows : p.rows);
  const long long tiles = (long long)c->kv_heads * ((rows + p.rows - 1) / p.rows);
  p.tiles = (int)(tiles < 0x7fffffff ? tiles : 0x7fffffff);
  const int ctas = (tc ? 1 : p.rows <= 8 ? 3 : 2) * sm_count;
  p.whole = !tc && a->max_kv_len <= 1024 && tiles * a->batch <= sm_count;
  p.workers = tc ? ctas : ctas * kWarps;
  p.by_tile = tiles * a->batch <= p.workers;
  p.records = p.by_tile ? p.tiles * a->batch : p.workers;
  auto bytes_of = [&](int workers, int rows) { return (size_t)workers * (sizeof(Kv8Record) + (size_t)2 * rows * (c->head_dim + 2) * sizeof(float)); };
  p.bytes = p.whole ? 0 : bytes_of(p.workers, p.rows);
  // what kv8_attention_tc_kernel takes suffices for the other one: so a call with smaller sizes never needs more
  if (rows > kFewRows) p.bytes = bytes_of(sm_count, kTcRows);
  return p;
}

template <int D, int TYPE, int ROWS, int WHOLE>
int launch(const Kv8AttnParams& ap, const Kv8AttnPlan& pl, const DeviceInfo* dev, cudaStream_t s) {
  using C = Cfg<D, ROWS, WHOLE>;
  static std::atomic<unsigned long long> allowed{0};
  int rc = allow_smem(kv8_attention_kernel<D, TYPE, ROWS, WHOLE>, C::kSmem, dev, allowed);
  if (rc != LIGER_OK) return rc;
  const dim3 grid = WHOLE ? dim3(pl.tiles, ap.e.batch) : dim3(pl.workers / kWarps);
  rc = launch_early("kv8_attention_kernel", kv8_attention_kernel<D, TYPE, ROWS, WHOLE>, grid, C::kThreads, C::kSmem, s, ap);
  return rc != LIGER_OK || WHOLE ? rc : launch_join<D, ROWS, kWarps>(ap, pl, dev, s);
}

template <int D, int TYPE>
int launch_rows(const Kv8AttnParams& ap, const Kv8AttnPlan& pl, const DeviceInfo* dev, cudaStream_t s) {
  switch (pl.rows) {
    case 4: return pl.whole ? launch<D, TYPE, 4, 1>(ap, pl, dev, s) : launch<D, TYPE, 4, 0>(ap, pl, dev, s);
    case 8: return pl.whole ? launch<D, TYPE, 8, 1>(ap, pl, dev, s) : launch<D, TYPE, 8, 0>(ap, pl, dev, s);
    case 16: return pl.whole ? launch<D, TYPE, 16, 1>(ap, pl, dev, s) : launch<D, TYPE, 16, 0>(ap, pl, dev, s);
    default: return pl.whole ? launch<D, TYPE, 24, 1>(ap, pl, dev, s) : launch<D, TYPE, 24, 0>(ap, pl, dev, s);
  }
}

int check_args(const liger_kv8_cache* c, const liger_kv8_attention_args* a) {
  if (!a) return set_error(LIGER_ERR_INVALID, "kv8_attention: args is NULL");
  int rc = kv8_check("kv8_attention", c, a->layer);
  if (rc != LIGER_OK) return rc;
  if (a->layer < 0) return set_error(LIGER_ERR_INVALID, "kv8_attention: layer %d", a->layer);
  if (a->heads <= 0 || a->heads % c->kv_heads)
    return set_error(LIGER_ERR_INVALID, "kv8_attention: heads = %d must be a positive multiple of kv_heads = %d", a->heads, c->kv_heads);
  rc = kv8_check_tokens("kv8_attention", a->q_offsets, a->batch, a->q_len, a->total_tokens, a->q_batch_stride, a->q_token_stride,
                        a->q_head_stride);
  if (rc != LIGER_OK) return rc;
  if ((long long)a->q_len * (a->heads / c->kv_heads) > (1 << 30))
    return set_error(LIGER_ERR_UNSUPPORTED, "kv8_attention: q_len * heads / kv_heads <= 2^30");
  if (a->max_kv_len < 0) return set_error(LIGER_ERR_INVALID, "kv8_attention: max_kv_len must not be negative");
  if (a->ldo % 8 || a->ldo < (long long)a->heads * c->head_dim)
    return set_error(LIGER_ERR_INVALID, "kv8_attention: ldo = %d must be a multiple of 8 and >= heads * head_dim = %lld", a->ldo,
                     (long long)a->heads * c->head_dim);
  return LIGER_OK;
}

// the SM count that workspaces are sized for where no device can be asked
constexpr int kAssumedSms = 148;

}  // namespace
}  // namespace liger

using namespace liger;

extern "C" size_t liger_kv8_attention_scratch_bytes(const liger_kv8_cache* cache, const liger_kv8_attention_args* args) {
  if (check_args(cache, args) != LIGER_OK) return 0;
  int dev = -1, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    sms = kAssumedSms;
  }
  return plan_of(cache, args, sms).bytes;
}

extern "C" int liger_kv8_attention(const liger_kv8_cache* cache, const liger_kv8_attention_args* a, void* stream) {
  int rc = check_args(cache, a);
  if (rc != LIGER_OK) return rc;
  if (!a->q || !a->out || !a->kv_lens) return set_error(LIGER_ERR_INVALID, "kv8_attention: a pointer is NULL");
  if (((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->scratch) & 15u)
    return set_error(LIGER_ERR_INVALID, "kv8_attention: q, out and scratch must be 16-byte aligned");
  if (((uintptr_t)a->kv_lens | (uintptr_t)a->slots) & 3u)
    return set_error(LIGER_ERR_INVALID, "kv8_attention: kv_lens and slots must be 4-byte aligned");
  if (!a->scratch && plan_of(cache, a, kAssumedSms).bytes) return set_error(LIGER_ERR_INVALID, "kv8_attention: scratch is NULL");
  const DeviceInfo* dev = nullptr;
  if ((rc = require_sm100(&dev)) != LIGER_OK) return rc;
  const Kv8AttnPlan pl = plan_of(cache, a, dev->sm_count);
  if (pl.bytes && !a->scratch) return set_error(LIGER_ERR_INVALID, "kv8_attention: scratch is NULL");
  if (a->scratch_bytes < pl.bytes)
    return set_error(LIGER_ERR_TOO_LARGE, "kv8_attention: scratch has %zu bytes, %zu are needed", a->scratch_bytes, pl.bytes);
  if (pl.tiles == 0x7fffffff) return set_error(LIGER_ERR_UNSUPPORTED, "kv8_attention: q_len %d x heads %d is too large", a->q_len, a->heads);
  Kv8AttnParams p{};
  p.c = kv8_layer(cache, a->layer);
  p.e = Kv8Entries{a->q_offsets, a->slots, a->batch, a->q_len, a->total_tokens};
  p.q = (const __half*)a->q;
  p.out = (__half*)a->out;
  p.kv_lens = a->kv_lens;
  p.q_batch_stride = a->q_batch_stride;
  p.q_token_stride = a->q_token_stride;
  p.q_head_stride = a->q_head_stride;
  p.heads = a->heads;
  p.group = a->heads / cache->kv_heads;
  p.max_kv_len = a->max_kv_len;
  p.ldo = a->ldo;
  p.causal = a->causal;
  p.scale_log2 = a->scale * kLog2e;
  p.tiles = pl.tiles;
  p.workers = pl.workers;
  p.by_tile = pl.by_tile;
  p.parts = (float*)a->scratch;
  p.records = (Kv8Record*)(p.parts + (size_t)2 * pl.workers * pl.rows * (cache->head_dim + 2));
  p.status = dev->status_dev;
  cudaStream_t s = (cudaStream_t)stream;
  if (pl.rows == kTcRows) return launch_kv8_attention_tc(p, pl, cache->head_dim, cache->type, dev, s);
  if (cache->head_dim == 128)
    return cache->type == LIGER_KV8_INT8 ? launch_rows<128, LIGER_KV8_INT8>(p, pl, dev, s) : launch_rows<128, LIGER_KV8_E4M3>(p, pl, dev, s);
  return cache->type == LIGER_KV8_INT8 ? launch_rows<64, LIGER_KV8_INT8>(p, pl, dev, s) : launch_rows<64, LIGER_KV8_E4M3>(p, pl, dev, s);
}
