// What the two kernels of attention over the paged 8-bit cache share: the call as the device sees it, equal shares of all
// sequences' work, and joining the parts of what lies across the border of two shares.
//
// Work is counted in places.  A tile (sequence, key head, row tile) has one for each step along its keys and a few for what it
// costs to begin one.  All tiles' places form one line, of which each worker (a warp or a CTA) takes an equal piece, whatever
// the sequences' lengths are.
#pragma once
#include "kv8.cuh"

namespace liger {

// A tile that is split, as the worker that begins it leaves it to the join.
struct alignas(16) Kv8Record {
  int first, last;          // the workers that have its first and its last part; first = -1: nothing to join
  int row0, row_base, rows; // the entry's first token, the tile's first row in the entry, the rows of the entry
  int head;
  int pad[2];
};

struct Kv8AttnParams {
  Kv8Layer c;
  Kv8Entries e;
  const __half* q;
  __half* out;
  const int* kv_lens;
  long long q_batch_stride, q_token_stride, q_head_stride;
  int heads, group, max_kv_len, ldo, causal;
  float scale_log2;
  int tiles;         // most tiles of an entry
  // shares
  int workers;       // warps or CTAs that share the work
  int by_tile;       // 1: records are numbered by entry and tile, 0: by the worker that began the tile
  Kv8Record* records;
  float* parts;      // [2 * workers] partial results
  DeviceStatus* status;
};


constexpr int kTcRows = 256;
// What a launch takes, as a function of a call's sizes and the SM count alone.
struct Kv8AttnPlan {
  int rows;      // rows of a tile; kTcRows: kv8_attention_tc_kernel
  int live;      // rows of a tile that can be in use
  int tiles;     // most tiles of an entry
  int whole;     // kv8_attention_kernel: a CTA takes a whole tile
  int workers, by_tile, records;
  size_t bytes;  // of scratch
};

// kv8_attention_sm100.cu
int launch_kv8_attention_tc(const Kv8AttnParams& p, const Kv8AttnPlan& pl, int head_dim, int type, const DeviceInfo* dev, cudaStream_t stream);

#ifdef __CUDACC__

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// An entry of the call with everything checked: n new tokens (rows row0 ..), len keys.  A bad length or slot gives len 0.
struct Entry {
  int n, row0, len, slot;
};
__device__ __forceinline__ Entry load_entry(const Kv8AttnParams& p, int b, bool report) {
  Entry e;
  if (!kv8_rows(p.e, b, e.n, e.row0) && report) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAttention, b, 0);
  e.len = kv8_ld(p.kv_lens + b);
  e.slot = kv8_slot(p.e, b);
  if (e.len < 0 || e.len > p.max_kv_len || e.slot < 0 || e.slot >= p.c.slots || e.len > ((long long)p.c.max_pages << p.c.page_shift)) {
    if (report) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAttention + 1, b, (unsigned)e.len);
    e.len = 0;
  }
  return e;
}
template <int ROWS>
__device__ __forceinline__ int row_tiles(const Kv8AttnParams& p, const Entry& e) { return (e.n * p.group + ROWS - 1) / ROWS; }

// a / b and a % b, by 32-bit division where that will do (a 64-bit one takes some 200 cycles)
__device__ __forceinline__ long long divide(long long a, int b, int& rest) {
  if ((unsigned long long)a >> 32 == 0) {
    const unsigned q = (unsigned)a / (unsigned)b;
    rest = (int)((unsigned)a - q * (unsigned)b);
    return q;
  }
  rest = (int)(a % b);
  return a / b;
}

// What a worker that begins a tile (first step of it) leaves for the join; `complete`: it also ends it.
__device__ __forceinline__ void leave_record(const Kv8AttnParams& p, int worker, bool complete, int last, const Entry& e, int b, int tile, int head,
                                             int row_base) {
  if (!p.by_tile && complete) return;
  int4* at = reinterpret_cast<int4*>(p.records + (p.by_tile ? (size_t)b * p.tiles + tile : (size_t)worker));
  at[0] = make_int4(complete ? -1 : worker, last, e.row0, row_base);
  at[1] = make_int4(e.n * p.group, head, 0, 0);
}

__device__ __forceinline__ int workers_used(long long total, int workers, int least) {
  int rest;
  const long long want = divide(total + least - 1, least, rest);
  return (int)(want < workers ? want : workers);
}
// How the line is dealt out: the first `more` workers have `each` + 1 places, the others `each`.
struct Kv8Deal {
  long long each;
  int more, used;
  __device__ __forceinline__ long long begin(int w) const { return each * w + min(w, more); }
  __device__ __forceinline__ int worker_of(long long at) const {
    int rest;
    const long long wide = (each + 1) * more;
    if (at < wide) return (int)(each + 1 < 0x7fffffff ? divide(at, (int)(each + 1), rest) : at / (each + 1));
    const int w = more + (int)(each < 0x7fffffff ? divide(at - wide, (int)each, rest) : (at - wide) / each);
    return min(w, used - 1);  // always, unless the lengths change under the call
  }
};

// Where the shares of a CTA's workers begin: entry and that entry's first place (entry -1: no share).
template <int SHARES>
struct Kv8Shares {
  Kv8Deal deal;
  int b[SHARES];
  long long first[SHARES];
};
// `line` gives the places of an entry; a share has at least `least`.  Ends with a barrier of the CTA.
template <int THREADS, int SHARES, typename Line>
__device__ __forceinline__ void find_shares(const Kv8AttnParams& p, int least, Line line, Kv8Shares<SHARES>& out) {
  constexpr int kW = THREADS / 32;
  __shared__ long long s_warp[kW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // most batches fit one round, whose places stay in registers
  const long long mine0 = threadIdx.x < p.e.batch ? line(load_entry(p, threadIdx.x, blockIdx.x == 0)) : 0;
  long long mine = mine0;
  for (int b = threadIdx.x + THREADS; b < p.e.batch; b += THREADS) mine += line(load_entry(p, b, blockIdx.x == 0));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_warp[warp] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) total += s_warp[w];
  Kv8Deal deal;
  deal.used = workers_used(total, p.workers, least);
  deal.each = divide(total, max(deal.used, 1), deal.more);
  if (threadIdx.x == 0) out.deal = deal;
  if (threadIdx.x < SHARES) out.b[threadIdx.x] = -1;
  __syncthreads();
  const int w0 = blockIdx.x * SHARES;
  if (w0 < deal.used) {
    const long long last = deal.begin(min(w0 + SHARES, deal.used) - 1);  // where the last of the CTA's shares begins
    long long before = 0;
    for (int base = 0; base < p.e.batch && before <= last; base += THREADS) {
      const int b = base + threadIdx.x;
      const long long v = base == 0 ? mine0 : b < p.e.batch ? line(load_entry(p, b, false)) : 0;
      long long incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) s_warp[warp] = incl;
      __syncthreads();
      long long all = 0;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        if (w < warp) incl += s_warp[w];
        all += s_warp[w];
      }
      const long long lo = before + incl - v, hi = before + incl;
#pragma unroll
      for (int w = 0; w < SHARES; ++w) {
        if (w0 + w >= deal.used) break;
        const long long at = deal.begin(w0 + w);
        if (at >= lo && at < hi) { out.b[w] = b; out.first[w] = lo; }
      }
      before += all;
      __syncthreads();
    }
  }
  __syncthreads();
}

// A value scale this much below the largest so far is taken for 0: in a result of fp16 such values do not show beside it.  The accumulators are
// in units of the reference scale, and so grow by no more than the inverse of this however often the reference moves.  With 2^9 for a code and sums of
// weights below 2^50 (2^28 keys of 2^15, and 2^16 for the reference score's way down, in kv8_attention_tc_kernel 2^59 in all) they stay below 2^128.
constexpr float kScaleVanishes = 8.6736174e-19f;  // 2^-60

constexpr int kJoinRowThreads = 256, kJoinThreads = 256;

// Joins the parts of the tiles that are split over several shares.  SHARED: a CTA has one row of a tile, whose parts its warps
// take in turn; else a warp has a row and takes all its parts.  Maxima, sums and accumulators of eight parts are fetched at once.
// GROUP workers in a row have joined their inner parts already (kv8_attention_kernel).  CTAs are small, so that they find room as the first
// kernel's leave: with 1024 threads instead of 256 a decode of 2 x 150001 tokens took 64 us instead of 59.
template <int D, int ROWS, int GROUP, int SHARED>
__global__ void __launch_bounds__(SHARED ? kJoinRowThreads : kJoinThreads) kv8_attention_join_kernel(const Kv8AttnParams p, int records, int live) {
  constexpr int kPart = ROWS * (D + 2);
  constexpr int kW = (SHARED ? kJoinRowThreads : kJoinThreads) / 32, kA = D / 32, kBatch = 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int which = SHARED ? blockIdx.x : blockIdx.x * kW + warp;  // record and row
  const int at = which / live, r = which % live;
  const int entry = at / p.tiles, tile = at % p.tiles;
  wait_for_stream();  // also for what the call before wrote, lengths and offsets: the first kernel's wait was for itself alone
  if (at >= records) return;
  const int4 rec = __ldcg(reinterpret_cast<const int4*>(p.records + at)), rec2 = __ldcg(reinterpret_cast<const int4*>(p.records + at) + 1);
  Entry e{};
  if (p.by_tile) kv8_rows(p.e, entry, e.n, e.row0);
  int row0 = rec.z, row = rec.w + r, rows = rec2.x, head = rec2.y;
  // nothing to join, or no two workers of this launch; the whole CTA where it shares a row
  if (rec.x < 0 || rec.y <= rec.x || rec.y >= p.workers || row >= rows) return;
  // the parts: the first worker's, those of workers between that begin a group, the last worker's
  const int begin = rec.x / GROUP, n = rec.y > rec.x ? (rec.y - 1) / GROUP - begin + 2 : 1;
  constexpr int kStride = SHARED ? kW : 1;
  float m = -INFINITY, l = 0.0f, a[kA];
#pragma unroll
  for (int i = 0; i < kA; ++i) a[i] = 0.0f;
  for (int i0 = SHARED ? warp : 0; i0 < n; i0 += kBatch * kStride) {
    float pm[kBatch], pl[kBatch], x[kBatch][kA];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int k = i0 + j * kStride;
      pm[j] = -INFINITY;
      pl[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < kA; ++i) x[j][i] = 0.0f;
      if (k < n) {
        // the first part is its worker's last tile, the others are their workers' first
        const float* q = p.parts + (size_t)(k == 0 ? 2 * rec.x + 1 : 2 * (k == n - 1 ? rec.y : (begin + k) * GROUP)) * kPart;
        pm[j] = __ldcg(q + r);
        pl[j] = __ldcg(q + ROWS + r);
        q += 2 * ROWS + r * D + lane * kA;
        if (D == 128) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(q));
          x[j][0] = v.x; x[j][1] = v.y; x[j][2 % kA] = v.z; x[j][3 % kA] = v.w;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(q));
          x[j][0] = v.x; x[j][1] = v.y;
        }
      }
    }
    float m_new = m;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m_new = fmaxf(m_new, pl[j] == 0.0f ? -INFINITY : pm[j]);
    // what saw nothing has no weight; a NaN stays
    const float fa = l == 0.0f ? 0.0f : l == l ? exp2_approx(m - m_new) : 1.0f;
    l *= fa;
#pragma unroll
    for (int i = 0; i < kA; ++i) a[i] *= fa;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float f = pl[j] == 0.0f ? 0.0f : pl[j] == pl[j] ? exp2_approx(pm[j] - m_new) : 1.0f;
      l = fmaf(f, pl[j], l);
#pragma unroll
      for (int i = 0; i < kA; ++i) a[i] = fmaf(f, x[j][i], a[i]);
    }
    m = m_new;
  }
  if (p.by_tile) {
    // A worker that gave up a wait leaves no record for the tiles that it did not reach, and the workspace holds anything: so what is written
    // to follows from the tile's number.  (Numbered by worker, every record is written by the launch that it belongs to.)  Asked for early and
    // looked at only here: in front of the parts it cost 0.4 us.
    const int tiles = row_tiles<ROWS>(p, e);
    if (tile >= p.c.kv_heads * tiles) return;
    row0 = e.row0;
    row = tile % tiles * ROWS + r;
    rows = e.n * p.group;
    head = tile / tiles;
    if (row >= rows) return;
  }
  const int token = row / p.group;
  __half* out = p.out + (size_t)(row0 + token) * p.ldo + (size_t)(head * p.group + row % p.group) * D;
  if (!SHARED) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (D == 128)
      *reinterpret_cast<uint2*>(out + lane * 4) = make_uint2(pack_half2(a[0] * inv, a[1] * inv), pack_half2(a[2 % kA] * inv, a[3 % kA] * inv));
    else
      *reinterpret_cast<uint32_t*>(out + lane * 2) = pack_half2(a[0] * inv, a[1] * inv);
    return;
  }
  __shared__ float s_m[kW], s_l[kW], s_a[kW][D];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int i = 0; i < kA; ++i) s_a[warp][lane * kA + i] = a[i];
  __syncthreads();
  if (threadIdx.x < D) {
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kW; ++w) mm = fmaxf(mm, s_l[w] == 0.0f ? -INFINITY : s_m[w]);
    float ll = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float f = s_l[w] == 0.0f ? 0.0f : s_l[w] == s_l[w] ? exp2_approx(s_m[w] - mm) : 1.0f;
      ll += f * s_l[w];
      y += f * s_a[w][threadIdx.x];
    }
    out[threadIdx.x] = __float2half_rn(ll == 0.0f ? 0.0f : y / ll);
  }
}

// Few tiles are split into many parts each: a CTA for each of their rows.
template <int D, int ROWS, int GROUP>
int launch_join(const Kv8AttnParams& ap, const Kv8AttnPlan& pl, const DeviceInfo* dev, cudaStream_t s) {
  const unsigned rows = (unsigned)pl.records * pl.live;
  if (rows <= 2u * dev->sm_count)
    return launch_early("kv8_attention_join_kernel", kv8_attention_join_kernel<D, ROWS, GROUP, 1>, dim3(rows), kJoinRowThreads, 0, s, ap, pl.records, pl.live);
  constexpr unsigned kRows = kJoinThreads / 32;
  return launch_early("kv8_attention_join_kernel", kv8_attention_join_kernel<D, ROWS, GROUP, 0>, dim3((rows + kRows - 1) / kRows), kJoinThreads, 0, s, ap,
                      pl.records, pl.live);
}

#endif

}  // namespace liger
