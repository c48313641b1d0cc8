// Attention over the paged 8-bit cache for many query rows per key head (a prompt, or a chunk of one, behind what the cache
// holds), on the tcgen05 tensor cores.
//
// What it cannot do without is tensor and exponential time, some 3100 and 2100 cycles for a block of 128 keys and 256 rows.  So
// a tile has 256 rows of one key head, two halves of 128 that take turns: while the softmax of one half runs, the products
// of the other do.  Rows are (new token, head of the group) pairs.
//
//   eight warps turn codes into fp16 (exact) and lay them down in shared memory the way the products read them (K with dims
//     contiguous, V as it lies, keys across; 128-byte swizzle), two blocks deep; the codes of the next block
//     wait in registers, its pages are looked up a block before that;  one warp works out the scales of each 16 keys;
//   two warps copy the queries of the next tile, half by half, as the last scores of this one are done;
//   one lane issues   S = Q K^T   (128 x 128, fp32 in TMEM)   and   O += P V   with P read from TMEM;
//   sixteen warps have half a row a thread: scores from TMEM, P = exp2 back into the place of S, as two fp16 parts; packed fp32 pairs.
// With five roles on one SM the instruction cache is what is short (a first form, unrolled throughout, missed it once in 28
// instructions and took three times as long): loops are kept rolled, and one warp walks the share for all.
//
// A key block's scale multiplies its columns of S in the same instruction that subtracts the reference score.  The value scale goes into
// the exponent, w = exp2(x - m + log2(scale / reference)), so that P V needs none; the row sum takes it out again, 16 columns
// at a time.  The reference is the first block's largest scale; O is rescaled where a block's largest leaves it (twice, a quarter).  The reference
// score follows the blocks' largest scores up and down (kAbove, kBelow), so that a block's weights do not fall out of fp16's range because
// another block's were larger: after a key that outweighs all others by 2^20 and whose value is small, the others make the result.  (That
// and the spills that came with it: 356 -> 363 us for the prompts below.)  P is a leading and a trailing fp16 part, like the other kernel's,
// and either is multiplied with V: one part alone, 2^-11 of each weight, shows in the result as much as the result's own rounding does
// (relative error of the prompts 2.89e-4 instead of 2.07e-4, 305 us instead of 356).  fp16 ends at 2^-24, so a weight is off by at most 2^-22 of
// itself or 2^-28 of the block's largest weight and value scale (where the reference score is as low as it goes: 2^-52 of the largest weight
// so far), whichever is more.
//
// Measured: 8 prompts of up to 512 tokens behind up to 2048, 96 heads of 128, int8: 363 us, 355 TFLOP/s (the trailing parts' products not
// counted).  With P in one part (305 us) a half's block took some 6400 cycles: 2000 .. 2500 until its scores were there (its O += P V and next S
// behind the other half's in one pipe; the trailing part of either half adds 512), 1100 .. 1400 for the maxima, 290 for telling the other warp,
// 2060 for the weights (the exponentials' own rate, when both halves are at it at once).  Tried with P in one part (then 331 us): scores of 64
// keys, computed one ahead, 348 us, since products of 64 columns cost as much time as those of 128; the weights handed over in two halves, no
// change; weights with the maximum so far in the same pass as the new one, 356 us: they have to wait in registers, and spill.
//
// Shares, parts and their joining: kv8_attention.cuh, a CTA being a worker and a block of 128 keys a step.
#include <type_traits>

#include "kv8_attention.cuh"

LIGER_REGISTER_WAIT_BUDGET()

namespace liger {
namespace {

constexpr int kBlock = 128;         // keys of a block, rows of a half
constexpr int kItemRows = kTcRows;
constexpr int kItemCost = 1;        // what it costs to begin a tile, in blocks (fitted to the CTAs' times: 1.5)
constexpr int kMinPlaces = 4;       // places that are worth a CTA
constexpr int kSoftmaxWarps = 16, kCodeWarps = 8, kQueryWarps = 2;
constexpr int kProductWarp = kSoftmaxWarps + kCodeWarps, kScaleWarp = kProductWarp + 1;
// Seven warpgroups of 72 registers a thread at launch, 896 * 72 in all; 512 * 80 + 256 * 56 + 128 * 72 is as much.
constexpr int kThreads = 896;
constexpr int kSoftmaxRegs = 80, kCodeRegs = 56, kProductRegs = 72;
constexpr int kBox = 128 * 128;     // 128 rows x 64 fp16
// Where the weights lie among fp16 numbers (in log2 units): the reference score has weight 2^11, a score up to 3 above it and a value scale up to
// twice the reference come on top.  A block's largest score is at most 6 below the reference score, unless that is 16 below the highest so far.
constexpr float kUnit = 11.0f, kAbove = 3.0f, kBelow = 6.0f, kLowest = 16.0f;
constexpr int kSlots = 4;           // scales of blocks

template <int D>
struct Cfg {
  static constexpr int kTile = D / 64 * kBox;
  static constexpr int kScaleBytes = kSlots * (8 * 16 + 16);
  static constexpr int kSmem = 6 * kTile /* Q x2, K x2, V x2 */ + kScaleBytes + 344 + 2 * 2 * 2 * 128 * 4 + 1024;
  static constexpr int kPart = kItemRows * (D + 2);
};

// Operand descriptors (fields: common.cuh).  Their upper halves are constants; an address, in units of 16 bytes, goes into the
// lower half.  Q and K: dims along the 128-byte rows.  V as B operand: dims along the rows, keys across them; the two boxes of
// 64 dims are kBox apart, groups of 8 keys 1024.
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  constexpr uint32_t kHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)kHigh << 32) | lo;
}
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t at) { return desc_of((at >> 4) | (1u << 16)); }
__device__ __forceinline__ uint64_t v_desc(uint32_t at) { return desc_of((at >> 4) | ((uint32_t)(kBox >> 4) << 16)); }
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 columns
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// waits for all loads so far; names the registers so that nothing uses them before
__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
// codes are read once: past L1, which is small here and holds what registers cannot
__device__ __forceinline__ uint4 load_code(const uint8_t* at) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
  return v;
}
__device__ __forceinline__ void sts32(uint32_t at, float x) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(x) : "memory"); }
__device__ __forceinline__ float lds32(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// a and b as fp16 and what that leaves of them, as fp16 again
__device__ __forceinline__ void two_parts(float a, float b, uint32_t& lead, uint32_t& trail) {
  lead = pack_half2(a, b);
  const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&lead));
  trail = pack_half2(a - back.x, b - back.y);
}

// ---- shared memory by 32-bit addresses: constants added to one register, where pointers would take two registers each --------------
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float4 lds128(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, float4 v) {
  sts128(at, __float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
}
// mbar_wait_bounded for a whole warp, with one answer for all lanes and fewer registers: the clock in steps of 2^16 ns.  Some warps wait for
// a whole tile, which takes as long as its keys are many; so the budget counts from the last time that the CTA's products went on (a number
// behind the abort flag), not from the wait's begin.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t abort_at) {
  uint32_t since = 0, seen = 0, done;
  for (uint32_t spins = 1;; ++spins) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) break;
    if ((spins & 0xffu) == 0) {
      uint32_t given_up, progress;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(given_up) : "r"(abort_at));
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(progress) : "r"(abort_at + 4));
      if (given_up) break;
      const uint32_t now = (uint32_t)(globaltimer_ns() >> 16);
      if (spins == 0x100u || progress != seen) {
        since = now;
        seen = progress;
      }
      if (now - since > (uint32_t)(g_wait_budget_ns >> 16) + 1u) {
        asm volatile("st.volatile.shared.u32 [%0], 1;" ::"r"(abort_at) : "memory");
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, done);
}

// Waits for products that have been issued, which end by themselves within microseconds; a million polls at most.
__device__ __forceinline__ void bar_drain(uint32_t bar) {
  for (uint32_t spins = 0, done = 0; !done && spins < (1u << 20); ++spins)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], 0;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar)
        : "memory");
}

// ---- the share of a CTA, tile by tile ---------------------------------------------------------------------------------------
struct Tile {
  int n0, n1;  // blocks that the halves see
  __device__ __forceinline__ int blocks() const { return max(n0, n1); }
  __device__ __forceinline__ int places() const { return max(1, blocks()) + kItemCost; }
};
// keys that row r of an entry sees
__device__ __forceinline__ int limit_of(const Kv8AttnParams& p, int len, int n, int r) {
  return p.causal ? min(len, max(0, len - n + r / p.group + 1)) : len;
}
__device__ __forceinline__ Tile tile_of(const Kv8AttnParams& p, const Entry& e, int rt) {
  const int rows = e.n * p.group, r0 = rt * kItemRows;
  Tile t;
  t.n0 = r0 < rows ? (limit_of(p, e.len, e.n, min(r0 + 127, rows - 1)) + kBlock - 1) / kBlock : 0;
  t.n1 = r0 + 128 < rows ? (limit_of(p, e.len, e.n, min(r0 + 255, rows - 1)) + kBlock - 1) / kBlock : 0;
  return t;
}
__device__ __forceinline__ int tiles_of(const Kv8AttnParams& p, const Entry& e) { return (e.n * p.group + kItemRows - 1) / kItemRows; }
__device__ __forceinline__ long long head_places(const Kv8AttnParams& p, const Entry& e) {
  const int tiles = tiles_of(p, e);
  if (!p.causal) return (long long)tiles * (tiles ? tile_of(p, e, 0).places() : 0);
  long long sum = 0;
  for (int i = 0; i < tiles; ++i) sum += tile_of(p, e, i).places();
  return sum;
}

struct Walk {
  long long at, end, tile0;  // places; tile0: the tile's first
  int b, head, rt, place;
  Entry e;
  Tile t;
  int s0, s1;                // blocks of this tile that are the share's: [s0, s1)
  int left;
  bool valid, first;         // first: the share began inside this tile
  __device__ __forceinline__ void cut(const Kv8AttnParams& p) {
    valid = at < end;
    if (!valid) return;
    t = tile_of(p, e, rt);
    const int places = t.places();
    left = (int)((long long)(places - place) < end - at ? places - place : end - at);
    tile0 = at - place;
    s0 = max(0, place - kItemCost);
    s1 = max(0, place + left - kItemCost);
  }
  __device__ __forceinline__ void start(const Kv8AttnParams& p, const Kv8Shares<1>& sh) {
    valid = sh.b[0] >= 0;
    if (!valid) return;
    at = sh.deal.begin(blockIdx.x);
    end = sh.deal.begin(blockIdx.x + 1);
    b = sh.b[0];
    e = load_entry(p, b, false);
    const long long inside = at - sh.first[0], per = head_places(p, e);
    head = min((int)(inside / per), p.c.kv_heads - 1);
    long long rest = inside % per;
    rt = 0;
    for (;;) {
      const int n = tile_of(p, e, rt).places();
      if (rest < n) break;
      rest -= n;
      ++rt;
    }
    place = (int)rest;
    first = true;
    cut(p);
  }
  __device__ __forceinline__ void next(const Kv8AttnParams& p) {
    at += left;
    place = 0;
    first = false;
    if (at < end && ++rt == tiles_of(p, e)) {
      rt = 0;
      if (++head == p.c.kv_heads) {
        head = 0;
        do {
          if (++b >= p.e.batch) {  // only if the lengths changed under the call
            valid = false;
            return;
          }
          e = load_entry(p, b, false);
        } while (e.n == 0);
      }
    }
    cut(p);
  }
  // blocks of half h in this share: [s0, stop(h))
  __device__ __forceinline__ int stop(int h) const { return max(s0, min(s1, h ? t.n1 : t.n0)); }
  __device__ __forceinline__ bool complete() const { return s0 == 0 && s1 == max(1, t.blocks()); }
};

// Pages and scales of a block: lane i has 16-key group i & 7, its page and its key scale (lanes 0 .. 7) or value scale (8 .. 15).
struct Lookup {
  const Kv8AttnParams& p;
  const int* row_table;
  int head, len, stop, page_mask, lane;
  __device__ __forceinline__ int page(int j) const {
    const int key = j * kBlock + (lane & 7) * 16;
    return lane < 16 && j < stop && key < len ? kv8_ld(row_table + (key >> p.c.page_shift)) : -1;
  }
  // -1 for a page that does not exist; told once, by the warp that has a status to tell
  __device__ __forceinline__ int valid(int page, int j, DeviceStatus* status, int b) const {
    if (page >= 0 && page < p.c.num_pages) return page;
    if (status && lane < 8 && j < stop && j * kBlock + lane * 16 < len) report_failure(status, LIGER_DEV_BAD_INDEX, kKv8AtAttention + 3, b, (unsigned)page);
    return -1;
  }
  __device__ __forceinline__ float scale(int page, int j) const {
    if (page < 0) return 0.0f;
    const int key = j * kBlock + (lane & 7) * 16;
    const size_t ph = (size_t)page * p.c.kv_heads + head;
    return kv8_ld((lane < 8 ? p.c.ks : p.c.vs) + (ph << (p.c.page_shift - p.c.block_shift)) + ((key & page_mask) >> p.c.block_shift));
  }
};

// What the warps need to know of a share's tile.  The scale warp walks the share and hands the tiles out in a ring: the walk is
// long code, and a copy of it in every role drove the kernel out of the instruction cache (170 KB, twice the time).
constexpr int kTiles = 4;
struct Segment {
  int valid;          // 0: the share ends
  int b, n, row0, len, slot, head, rt;
  int s0, s1;         // blocks [s0, s1); s1 = 0: the share ends before the tile's first block
  int stop0, stop1;   // where the halves stop
  int complete;       // the whole tile is this share's
  int part;           // where its part goes, if it is not
};

template <int D, int TYPE>
__global__ void __launch_bounds__(kThreads, 1) kv8_attention_tc_kernel(const Kv8AttnParams p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sQ = (smem_u32(smem_raw) + 1023u) & ~1023u;  // [2]
  const uint32_t sK = sQ + 2 * C::kTile;                      // [2]
  const uint32_t sV = sK + 2 * C::kTile;                      // [2]
  const uint32_t s_scale = sV + 2 * C::kTile;                 // [slots][8] float4: key scale, log2 of value scale, its inverse (-1: 0), mask
  const uint32_t s_ref = s_scale + kSlots * 8 * 16;           // [slots] float4: reference, old reference / new one, not plain
  const uint32_t bars = s_ref + kSlots * 16;
  const uint32_t q_full = bars, q_empty = bars + 16;          // [2] each: halves
  const uint32_t k_full = bars + 32, k_empty = bars + 48;     // [2]: stages
  const uint32_t v_full = bars + 64, v_empty = bars + 80;
  const uint32_t s_full = bars + 96, p_full = bars + 112;     // [2]: halves
  const uint32_t o_full = bars + 128, o_empty = bars + 144;
  const uint32_t sc_full = bars + 160;                        // [slots]
  const uint32_t t_full = bars + 192, t_empty = bars + 224;   // [kTiles]
  const uint32_t tmem_slot = bars + 256, abort_flag = bars + 260, progress = bars + 264;  // of the products, for bar_wait: behind the flag
  const uint32_t pairs = bars + 272;                          // [8]: two warps that share 32 rows
  const uint32_t drained = bars + 336;                        // products that are under way as the CTA gives up
  const uint32_t s_pair = bars + 344;                         // [maxima, sums][half][half of the keys][128 rows]
  __shared__ Kv8Shares<1> shares;
  __shared__ Segment segments[kTiles];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(q_full + i * 8, kQueryWarps);
      bar_init(q_empty + i * 8, 1);
      bar_init(k_full + i * 8, kCodeWarps + 1);  // K and its scales
      bar_init(k_empty + i * 8, 1);
      bar_init(v_full + i * 8, kCodeWarps);
      bar_init(v_empty + i * 8, 1);
      bar_init(s_full + i * 8, 1);
      bar_init(p_full + i * 8, kSoftmaxWarps / 2);
      bar_init(o_full + i * 8, 1);
      bar_init(o_empty + i * 8, kSoftmaxWarps / 2);
    }
    for (int i = 0; i < kSlots; ++i) bar_init(sc_full + i * 8, 1);
    for (int i = 0; i < kTiles; ++i) {
      bar_init(t_full + i * 8, 1);
      bar_init(t_empty + i * 8, kThreads / 32);
    }
    for (int i = 0; i < 8; ++i) bar_init(pairs + i * 8, 2);
    bar_init(drained, 1);
    asm volatile("st.volatile.shared.u32 [%0], 0;" ::"r"(abort_flag) : "memory");
    asm volatile("st.volatile.shared.u32 [%0], 0;" ::"r"(progress) : "memory");
    fence_barrier_init();
  }
  if (warp == kProductWarp) {
    // S at columns 0 / 128, O at 256 / 384
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
    tmem_relinquish();
  }
  tc_fence_before();
  wait_for_stream();
  find_shares<kThreads>(p, kMinPlaces, [&](const Entry& x) { return (long long)p.c.kv_heads * head_places(p, x); }, shares);
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  const int worker = blockIdx.x;
  // the next tile of the share; false at its end.  A warp gives a tile back when it asks for the next one.
  uint32_t tiles_had = 0;
  auto next_tile = [&]() -> const Segment* {
    if (tiles_had) {
      __syncwarp();
      if (lane == 0) bar_arrive(t_empty + ((tiles_had - 1) & 3u) * 8);
    }
    const uint32_t i = tiles_had & 3u;
    if (!bar_wait(t_full + i * 8, (tiles_had >> 2) & 1u, abort_flag)) return nullptr;
    ++tiles_had;
    return segments[i].valid ? &segments[i] : nullptr;
  };

  if (warp >= kSoftmaxWarps && warp < kProductWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCodeRegs));
    // ===== codes -> fp16 tiles, scales =====
    const int cw = warp - kSoftmaxWarps;
    constexpr int kChunks = D / 16, kKeysPass = kCodeWarps * 32 / kChunks, kPass = kBlock / kKeysPass;
    // lane quads have neighbouring chunks of a key, neighbouring quads neighbouring keys: no two store to one bank
    const int c = D == 128 ? (lane & 3) + ((lane >> 3) & 1) * 4 : lane & 3;
    const int r_in = D == 128 ? cw * 4 + ((lane >> 2) & 1) + (lane >> 4) * 2 : cw * 8 + (lane >> 2);
    const int group_in = r_in >> 4;  // of 16 keys, inside a pass
    const int page_mask = (1 << p.c.page_shift) - 1;
    uint32_t g = 0;
    bool ok = true;
    while (ok) {
      const Segment* w = next_tile();
      if (!w) break;
      const int s0 = w->s0, stop = max(w->stop0, w->stop1), len = w->len, head = w->head;
      if (stop <= s0) continue;
      const int* row_table = p.c.table + (size_t)w->slot * p.c.max_pages;
      const Lookup look{p, row_table, head, len, stop, page_mask, lane};
      auto load = [&](const uint8_t* base, int j, int pages, uint4 (&x)[kPass]) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          const int key = j * kBlock + i * kKeysPass + r_in;
          const int page = __shfl_sync(0xffffffffu, pages, (i * kKeysPass >> 4) + group_in);
          x[i] = make_uint4(0, 0, 0, 0);
          if (page >= 0 && key < len)
            x[i] = load_code(base + ((((size_t)page * p.c.kv_heads + head) << p.c.page_shift) + (key & page_mask)) * D + c * 16);
        }
      };
      auto store = [&](uint32_t tile, const uint4 (&x)[kPass]) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          const int r = i * kKeysPass + r_in;
          const uint32_t row = tile + (c >> 2) * kBox + r * 128;
          const int idx = (c & 3) * 2;
          const uint32_t a = kv8_bias<TYPE>(x[i].x), b = kv8_bias<TYPE>(x[i].y), d = kv8_bias<TYPE>(x[i].z), e = kv8_bias<TYPE>(x[i].w);
          sts128(row + ((idx ^ (r & 7)) << 4), kv8_pair<TYPE, 0>(a), kv8_pair<TYPE, 1>(a), kv8_pair<TYPE, 0>(b), kv8_pair<TYPE, 1>(b));
          sts128(row + (((idx + 1) ^ (r & 7)) << 4), kv8_pair<TYPE, 0>(d), kv8_pair<TYPE, 1>(d), kv8_pair<TYPE, 0>(e), kv8_pair<TYPE, 1>(e));
        }
      };
      // The fence between these writes and the tensor core's reads is the product warp's, after its wait: here it would also wait
      // for the loads of the next block that are under way.
      auto publish = [&](uint32_t bar) {
        __syncwarp();
        if (lane == 0) bar_arrive(bar);
      };

      // Half rounds: K of block j, V of block j, K of block j + 1, ..., each laid down and then the next one's codes fetched; the
      // pages of a block are looked up a block ahead.  One copy of the code for both, since the instruction cache is what is short.
      uint4 x[kPass];
      int page_now = look.valid(look.page(s0), s0, nullptr, 0), page_next = look.page(s0 + 1);
      load(p.c.k, s0, page_now, x);
#pragma unroll 1
      for (int i = 2 * s0; i < 2 * stop; ++i) {
        const uint32_t is_v = i & 1u, st = g & 1u, ph = (g >> 1) & 1u;
        if (!bar_wait((is_v ? v_empty : k_empty) + st * 8, ph ^ 1u, abort_flag)) { ok = false; break; }
        store((is_v ? sV : sK) + st * C::kTile, x);
        publish((is_v ? v_full : k_full) + st * 8);
        const int j = (i + 1) >> 1;
        if (is_v) {
          ++g;
          page_now = look.valid(page_next, j, nullptr, 0);
          page_next = look.page(j + 1);
        }
        load(is_v ? p.c.k : p.c.v, j, page_now, x);
      }
    }
  } else if (warp >= kProductWarp) {
    // ===== products =====
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProductRegs));
    if (warp == kProductWarp) {
      // The whole warp walks and waits, one elected lane issues: then the compiler knows that the descriptors are the same for
      // all lanes that run, and an issue costs a few cycles; inside `if (lane == 0)` it cost over 200.
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128);
      constexpr uint32_t idesc_o = make_idesc_f16(128, D) | (1u << 16);  // B with dims contiguous
      uint32_t g = 0, nq = 0, np = 0, no = 0;  // parities of what the halves have had: bit h
      bool ok = true;
      while (ok) {
        const Segment* w = next_tile();
        if (!w) break;
        const int s0 = w->s0, e0 = w->stop0, e1 = w->stop1, stop = max(e0, e1);
        if (stop <= s0) continue;
        // round j: O += P V of block j, then S of block j + 1, for one half and the other (round s0 - 1: S only)
#pragma unroll 1
        for (int j = s0 - 1; j < stop && ok; ++j) {
          const uint32_t n = g + (uint32_t)(j - s0);
          // the tiles first, so that nothing but the weights stands between them and the products
          if ((j >= s0 && !bar_wait(v_full + (n & 1u) * 8, (n >> 1) & 1u, abort_flag)) ||
              (j + 1 < stop && !bar_wait(k_full + ((n + 1) & 1u) * 8, ((n + 1) >> 1) & 1u, abort_flag))) { ok = false; break; }
          fence_proxy_async();  // V, K
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const int end = h ? e1 : e0;
            if (j >= s0 && j < end) {
              const uint32_t st = n & 1u;
              if (!bar_wait(p_full + h * 8, (np >> h) & 1u, abort_flag) || (j == s0 && !bar_wait(o_empty + h * 8, ((no >> h) & 1u) ^ 1u, abort_flag))) { ok = false; break; }
              np ^= 1u << h;
              if (j == s0) no ^= 1u << h;
              tc_fence_after();
              if (elect_one()) {
                const uint32_t va = sV + st * C::kTile, o = tmem + 256 + h * 128, pa = tmem + h * 128;
#pragma unroll
                for (int k = 0; k < 8; ++k) {  // 16 keys each, both parts of their weights
                  umma_f16_ts(o, pa + k * 16, v_desc(va + k * 2048), idesc_o, (j != s0 || k != 0) ? 1u : 0u);
                  umma_f16_ts(o, pa + k * 16 + 8, v_desc(va + k * 2048), idesc_o, 1u);
                }
                if (j == end - 1) bar_commit(o_full + h * 8);
              }
              __syncwarp();
            }
            if (j + 1 < end) {
              const uint32_t m = n + 1, st = m & 1u;
              if (j < s0) {
                if (!bar_wait(q_full + h * 8, (nq >> h) & 1u, abort_flag)) { ok = false; break; }
                nq ^= 1u << h;
                fence_proxy_async();
              }
              tc_fence_after();
              if (elect_one()) {
                const uint32_t qa = sQ + h * C::kTile, ka = sK + st * C::kTile;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                  const uint64_t da = kmajor_desc(qa + (k >> 2) * kBox + (k & 3) * 32), db = kmajor_desc(ka + (k >> 2) * kBox + (k & 3) * 32);
                  umma_f16(tmem + h * 128, da, db, idesc_s, k != 0 ? 1u : 0u);
                }
                bar_commit(s_full + h * 8);
                if (j + 1 == end - 1) bar_commit(q_empty + h * 8);
              }
              __syncwarp();
            }
          }
          if (!ok) break;
          if (elect_one()) {
            asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(progress), "r"(n + 2u) : "memory");
            if (j >= s0) bar_commit(v_empty + (n & 1u) * 8);
            if (j + 1 < stop) bar_commit(k_empty + ((n + 1) & 1u) * 8);
          }
          __syncwarp();
        }
        g += (uint32_t)(stop - s0);
      }
    } else if (warp == kScaleWarp) {
      // ===== the walk, and the scales of the blocks' eight groups =====
      uint32_t g = 0, given = 0;
      bool ok = true;
      Walk walk;
      walk.start(p, shares);
      if (!p.by_tile && lane == 0) p.records[worker].first = -1;
      // hands the walk's tile out and goes on to the next
      auto hand_out = [&]() {
        const uint32_t i = given & 3u;
        if (!bar_wait(t_empty + i * 8, ((given >> 2) & 1u) ^ 1u, abort_flag)) { ok = false; return; }
        ++given;
        if (lane == 0) {
          Segment s;
          s.valid = walk.valid;
          if (walk.valid) {
            s.b = walk.b; s.n = walk.e.n; s.row0 = walk.e.row0; s.len = walk.e.len; s.slot = walk.e.slot;
            s.head = walk.head; s.rt = walk.rt; s.s0 = walk.s0; s.s1 = walk.s1; s.stop0 = walk.stop(0); s.stop1 = walk.stop(1);
            s.complete = walk.complete();
            s.part = 2 * worker + (walk.first && walk.s0 > 0 ? 0 : 1);
            if (s.s0 == 0 && s.s1 > 0)  // who begins a tile knows who ends it
              leave_record(p, worker, s.complete, s.complete ? 0 : shares.deal.worker_of(walk.tile0 + walk.t.places() - 1), walk.e, s.b,
                           s.head * tiles_of(p, walk.e) + s.rt, s.head, s.rt * kItemRows);
          }
          segments[i] = s;
        }
        __syncwarp();
        if (lane == 0) bar_arrive(t_full + i * 8);
        if (walk.valid) walk.next(p);
      };
      bool more = walk.valid;
      hand_out();
      while (ok) {
        if (more) {  // one ahead of what this warp works on; the end of the share is a tile, too
          more = walk.valid;
          hand_out();
          if (!ok) break;
        }
        const Segment* w = next_tile();
        if (!w) break;
        const int s0 = w->s0, stop = max(w->stop0, w->stop1), b = w->b;
        if (stop <= s0) continue;
        const Lookup look{p, p.c.table + (size_t)w->slot * p.c.max_pages, w->head, w->len, stop, (1 << p.c.page_shift) - 1, lane};
        int page_now = look.valid(look.page(s0), s0, p.status, b), page_next = look.page(s0 + 1);
        float scale_now = look.scale(page_now, s0), ref = 0.0f, ref_top = 0.0f;
        for (int j = s0; j < stop; ++j, ++g) {
          page_next = look.valid(page_next, j + 1, p.status, b);
          const float scale_next = look.scale(page_next, j + 1);
          const int page_after = look.page(j + 2);
          // a slot is free when K's stage is: by then both halves are past the block before the last
          if (!bar_wait(k_empty + (g & 1u) * 8, ((g >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
          // scales of the block's eight groups: lanes 0 .. 7
          const float mine = scale_now >= 0.0f && scale_now < INFINITY ? scale_now : NAN;
          const float vs = __shfl_sync(0xffffffffu, mine, (lane & 7) + 8);
          const bool use = lane < 8 && page_now >= 0 && vs > 0.0f;
          const float top = warp_max(use ? vs : 0.0f);
          float moved = 1.0f;
          if (ref == 0.0f) {
            ref = top;
          } else if (top > ref * 2.0f || (top < ref * 0.25f && top > ref_top * kScaleVanishes)) {
            moved = ref / top;
            ref = top;
          }
          ref_top = fmaxf(ref_top, ref);
          const float base = ref > 0.0f ? ref : 1.0f;
          const bool vanishes = page_now >= 0 && vs <= base * kScaleVanishes;
          if (lane < 8)
            sts128(s_scale + ((g & 3u) * 8 + lane) * 16,
                   make_float4(page_now >= 0 ? mine * p.scale_log2 : 0.0f,
                               page_now < 0 ? -INFINITY : vanishes ? 0.0f : vs > 0.0f ? __log2f(vs / base) : NAN,
                               vanishes ? -1.0f : use ? base / vs : 1.0f, page_now < 0 ? -INFINITY : 0.0f));
          // scales that vanish or are not finite, pages that are missing: such a block is weighed with care
          const bool odd = __any_sync(0xffffffffu, lane < 16 && (!(mine > 0.0f) || (lane < 8 && vanishes)));
          if (lane == 0) sts128(s_ref + (g & 3u) * 16, make_float4(base, moved, odd ? 1.0f : 0.0f, 0.0f));
          __syncwarp();
          if (lane == 0) {
            bar_arrive(sc_full + (g & 3u) * 8);
            bar_arrive(k_full + (g & 1u) * 8);  // no score before its scale: so this warp cannot fall two stages behind
          }
          page_now = page_next;
          scale_now = scale_next;
          page_next = page_after;
        }
      }
    } else {
      // ===== queries =====
      const int qt = threadIdx.x - (kScaleWarp + 1) * 32;
      constexpr int kQChunks = D / 8;
      uint32_t nq[2] = {0, 0};
      bool ok = true;
      while (ok) {
        const Segment* w = next_tile();
        if (!w) break;
        const int rows = w->n * p.group;
        const __half* base = p.q + (p.e.q_offsets ? (long long)w->row0 * p.q_token_stride : (long long)w->b * p.q_batch_stride) +
                             (long long)w->head * p.group * p.q_head_stride;
#pragma unroll 1
        for (int h = 0; h < 2 && ok; ++h) {
          if ((h ? w->stop1 : w->stop0) <= w->s0) continue;
          if (!bar_wait(q_empty + h * 8, (nq[h] & 1u) ^ 1u, abort_flag)) { ok = false; break; }
          ++nq[h];
          const int r0 = w->rt * kItemRows + h * 128;
          // a thread has one 16-byte piece of every kStep-th row; row r is token r / group, head r % group
          constexpr int kStep = kQueryWarps * 32 / kQChunks;
          const int qc = qt % kQChunks;
          int r = r0 + qt / kQChunks, hh = r % p.group;
          const __half* src = base + (long long)(r / p.group) * p.q_token_stride + (long long)hh * p.q_head_stride + qc * 8;
          const int d_token = kStep / p.group, d_hh = kStep - d_token * p.group;
          const long long d_src = d_token * p.q_token_stride + d_hh * p.q_head_stride, d_wrap = p.q_token_stride - p.group * p.q_head_stride;
          uint32_t dst = sQ + h * C::kTile + (qc >> 3) * kBox + (r & 127) * 128;
#pragma unroll 4
          for (int i = 0; i < 128 / kStep; ++i) {
            const bool there = r < rows;  // rows that are not there are zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (((qc & 7) ^ (r & 7)) << 4)), "l"(there ? src : p.q),
                         "r"(there ? 16 : 0)
                         : "memory");
            r += kStep;
            dst += kStep * 128;
            src += d_src;
            hh += d_hh;
            if (hh >= p.group) {
              hh -= p.group;
              src += d_wrap;
            }
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
          if (lane == 0) bar_arrive(q_full + h * 8);
        }
      }
    }
  } else {
    // ===== softmax and output: thread = row of half h, half `cp` of a block's keys and of the output's dims =====
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int h = warp >> 3, cp = (warp >> 2) & 1, quad = warp & 3;
    const int r_tile = h * 128 + quad * 32 + lane, pair = h * 4 + quad;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + h * 128 + cp * 64 + lanes;
    const uint32_t o_addr = tmem + 256 + h * 128 + cp * (D / 2) + lanes;
    const uint32_t mine = s_pair + ((h * 2 + cp) * 128 + quad * 32 + lane) * 4, others = mine + (cp ? -512 : 512);
    uint32_t g = 0, ns = 0, no = 0, met = 0;
    bool ok = true;
    // waits for the pair's other warp: either sees what the other has written
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) bar_arrive(pairs + pair * 8);
      const bool there = bar_wait(pairs + pair * 8, met & 1u, abort_flag);
      ++met;
      return there;
    };
    while (ok) {
      const Segment* w = next_tile();
      if (!w) break;
      if (w->s1 == 0) continue;
      const int s0 = w->s0, stop = h ? w->stop1 : w->stop0, all = max(w->stop0, w->stop1);
      const int rows = w->n * p.group, r = w->rt * kItemRows + r_tile;
      const int limit = r < rows ? limit_of(p, w->len, w->n, r) : 0;
      // rows that are not there ask for no mask: the last tile of a prompt would else take the careful way throughout (332 -> 307 us)
      const int limit_low = __reduce_min_sync(0xffffffffu, r < rows ? limit : w->len), limit_high = __reduce_max_sync(0xffffffffu, limit);
      float m_ref = -INFINITY, m_top = -INFINITY, l = 0.0f, ref = 1.0f;
#pragma unroll 1
      for (int j = s0; j < stop; ++j, ++ns) {
        const uint32_t n = g + (uint32_t)(j - s0), slot = n & 3u;
        if (!bar_wait(sc_full + slot * 8, (n >> 2) & 1u, abort_flag) || !bar_wait(s_full + h * 8, ns & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t sc = s_scale + slot * 128 + cp * 64;
        const float4 rf = lds128(s_ref + slot * 16);
        ref = rf.x;
        const int cut = limit - j * kBlock - cp * 64;  // this thread's columns from here on are not seen
        // groups of 16 columns: the first `free` are seen by all rows of the warp (none, where a page is missing or a scale is 0 or not
        // finite), those from `shut` on by none
        const int shut = min(4, (limit_high - j * kBlock - cp * 64 + 15) >> 4);
        const int free = rf.z == 0.0f ? min(shut, (limit_low - j * kBlock - cp * 64) >> 4) : 0;
        // the rows' largest scores, in log2 units and without the value scales; the two warps of a row tell each other
        float mx = -INFINITY;
#pragma unroll 1
        for (int gi = 0; gi < shut; ++gi) {
          uint32_t x[16];
          tmem_ld_32x16(s_addr + gi * 16, x);
          const float4 f = lds128(sc + gi * 16);
          float a = -INFINITY, b = -INFINITY;
          tmem_ld_wait16(x);
          if (gi < free) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              a = fmaxf(a, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
              b = fmaxf(b, fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
            }
          } else {
            const int seen = cut - gi * 16;
#pragma unroll
            for (int i = 0; i < 16; ++i) a = i < seen ? fmaxf(a, __uint_as_float(x[i])) : a;
          }
          a = fmaxf(a, b);
          mx = fmaxf(mx, a == -INFINITY ? a : fmaf(a, f.x, f.w));
        }
        sts32(mine, mx);
        if (!meet()) { ok = false; break; }
        mx = fmaxf(mx, lds32(others));
        float m_try = m_ref;
        if (mx > m_ref + kAbove || (mx < m_ref - kBelow && mx > -INFINITY)) {
          m_try = fmaxf(mx, m_top - kLowest);
          m_top = fmaxf(m_top, m_try);
        }
        const float m_safe = m_try == -INFINITY ? 0.0f : m_try - kUnit;
        // the weights, 16 keys at a time; their leading and trailing parts take the place of the scores that they come from
        float sum = 0.0f;
#pragma unroll 1
        for (int gi = 0; gi < 4; ++gi) {
          uint32_t pk[16];  // leading, trailing parts
          if (gi >= shut) {
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = 0;
          } else {
            uint32_t x[16];
            tmem_ld_32x16(s_addr + gi * 16, x);
            const float4 f = lds128(sc + gi * 16);
            const float off = f.y - m_safe;
            tmem_ld_wait16(x);
            float total;
            if (gi < free) {
              const uint64_t f2 = pack2(f.x, f.x), off2 = pack2(off, off);
              uint64_t a = 0, b = 0;
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float2 y0 = unpack2(fma2(pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), f2, off2));
                const float2 y1 = unpack2(fma2(pack2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), f2, off2));
                const float w0 = exp2_approx(y0.x), w1 = exp2_approx(y0.y), w2 = exp2_approx(y1.x), w3 = exp2_approx(y1.y);
                a = add2(a, pack2(w0, w1));
                b = add2(b, pack2(w2, w3));
                two_parts(w0, w1, pk[i >> 1], pk[(i >> 1) + 8]);
                two_parts(w2, w3, pk[(i >> 1) + 1], pk[(i >> 1) + 9]);
              }
              const float2 ab = unpack2(add2(a, b));
              total = ab.x + ab.y;
            } else {
              const int seen = cut - gi * 16;
              total = 0.0f;
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                float w0 = exp2_approx(fmaf(__uint_as_float(x[i]), f.x, off)), w1 = exp2_approx(fmaf(__uint_as_float(x[i + 1]), f.x, off));
                w0 = i < seen ? w0 : 0.0f;
                w1 = i + 1 < seen ? w1 : 0.0f;
                total += w0 + w1;
                two_parts(f.z < 0.0f ? 0.0f : w0, f.z < 0.0f ? 0.0f : w1, pk[i >> 1], pk[(i >> 1) + 8]);  // values of zero scale are zeros whatever their codes are
              }
            }
            sum = fmaf(total, fabsf(f.z), sum);
          }
          tmem_st_32x16(s_addr + gi * 16, pk);
        }
        float alpha = rf.y;
        if (m_try != m_ref) {
          const float shrink = m_ref == -INFINITY ? 0.0f : exp2_approx(m_ref - m_try);
          alpha *= shrink;
          l *= shrink;
          m_ref = m_try;
        }
        l += sum;
        if (j > s0 && __any_sync(0xffffffffu, alpha != 1.0f)) {  // the products so far are complete: S came after them
#pragma unroll 1
          for (int ch = 0; ch < D / 64; ++ch) {
            uint32_t v[32];
            tmem_ld_32x32(o_addr + ch * 32, v);
            tmem_ld_wait_regs(v);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
            tmem_st_32x32(o_addr + ch * 32, v);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(p_full + h * 8);
      }
      if (!ok) break;
      g += (uint32_t)(all > s0 ? all - s0 : 0);
      // the row's result, or its part
      const bool some = stop > s0, complete = w->complete;
      if (some) {
        sts32(mine + 2048, l);
        if (!meet()) { ok = false; break; }
        l += lds32(others + 2048);
        if (!bar_wait(o_full + h * 8, no & 1u, abort_flag)) { ok = false; break; }
        ++no;
        tc_fence_after();
      }
      const float inv = l == 0.0f ? 0.0f : ref / l;
      const int token = r / p.group;
      __half* out = p.out + (size_t)(w->row0 + token) * p.ldo + (size_t)(w->head * p.group + r % p.group) * D + cp * (D / 2);
      float* part = p.parts + (size_t)w->part * C::kPart;
      if (!complete && r < rows && cp == 0) { part[r_tile] = m_ref; part[kItemRows + r_tile] = l; }
      part += 2 * kItemRows + (size_t)r_tile * D + cp * (D / 2);
#pragma unroll 1
      for (int ch = 0; ch < D / 64; ++ch) {
        uint32_t v[32];
        if (some) {
          tmem_ld_32x32(o_addr + ch * 32, v);
          tmem_ld_wait_regs(v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (r < rows) {
          if (complete) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(out + ch * 32 + i * 8) =
                  make_uint4(pack_half2(__uint_as_float(v[i * 8]) * inv, __uint_as_float(v[i * 8 + 1]) * inv),
                             pack_half2(__uint_as_float(v[i * 8 + 2]) * inv, __uint_as_float(v[i * 8 + 3]) * inv),
                             pack_half2(__uint_as_float(v[i * 8 + 4]) * inv, __uint_as_float(v[i * 8 + 5]) * inv),
                             pack_half2(__uint_as_float(v[i * 8 + 6]) * inv, __uint_as_float(v[i * 8 + 7]) * inv));
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float4*>(part + ch * 32 + i * 4) = make_float4(__uint_as_float(v[i * 4]) * ref, __uint_as_float(v[i * 4 + 1]) * ref,
                                                                               __uint_as_float(v[i * 4 + 2]) * ref, __uint_as_float(v[i * 4 + 3]) * ref);
          }
        }
      }
      if (some) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(o_empty + h * 8);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  uint32_t given_up;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(given_up) : "r"(abort_flag));
  if (warp == kProductWarp) {
    tc_fence_after();
    if (given_up) {  // nobody may have waited for the last products: they end before the memory that they use goes to others
      if (elect_one()) bar_commit(drained);
      __syncwarp();
      bar_drain(drained);
    }
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && given_up) report_failure(p.status, LIGER_DEV_TIMEOUT, 0x210u, blockIdx.x, 0);
}

template <int D, int TYPE>
int launch(const Kv8AttnParams& p, const Kv8AttnPlan& pl, const DeviceInfo* dev, cudaStream_t s) {
  static std::atomic<unsigned long long> allowed{0};
  int rc = allow_smem(kv8_attention_tc_kernel<D, TYPE>, Cfg<D>::kSmem, dev, allowed);
  if (rc != LIGER_OK) return rc;
  rc = launch_early("kv8_attention_tc_kernel", kv8_attention_tc_kernel<D, TYPE>, dim3(pl.workers), kThreads, Cfg<D>::kSmem, s, p);
  return rc != LIGER_OK ? rc : launch_join<D, kItemRows, 1>(p, pl, dev, s);
}

}  // namespace

int launch_kv8_attention_tc(const Kv8AttnParams& p, const Kv8AttnPlan& pl, int head_dim, int type, const DeviceInfo* dev, cudaStream_t s) {
  if (head_dim == 128) return type == LIGER_KV8_INT8 ? launch<128, LIGER_KV8_INT8>(p, pl, dev, s) : launch<128, LIGER_KV8_E4M3>(p, pl, dev, s);
  return type == LIGER_KV8_INT8 ? launch<64, LIGER_KV8_INT8>(p, pl, dev, s) : launch<64, LIGER_KV8_E4M3>(p, pl, dev, s);
}

}  // namespace liger
