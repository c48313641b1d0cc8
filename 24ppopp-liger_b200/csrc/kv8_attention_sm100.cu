// Attention over the paged 8-bit cache for many query rows per key head (a prompt, or a chunk of one, behind what the cache
// holds), on the tcgen05 tensor cores.
//
// Bound by the tensor pipe and, as closely, by the exponentials: a block of 128 keys costs 256 rows 2048 cycles of either.  So
// a tile has 256 rows of one key head, two halves of 128 that take turns: while the softmax of one half runs, the products
// of the other do.  Rows are (new token, head of the group) pairs.
//
//   eight warps turn codes into fp16 (exact) and lay them down in shared memory the way the products read them (K with dims
//     contiguous, V as it lies, keys across; 128-byte swizzle), two blocks deep, and work out each 16 keys' scales; the codes
//     of the next block wait in registers, its pages and scales are looked up a block before that;
//   three warps copy the queries of the next tile, half by half, as the last scores of this one are done;
//   one lane issues   S = Q K^T   (128 x 128, fp32 in TMEM)   and   O += P V   with P read from TMEM;
//   eight warps have a row a thread: scores from TMEM, P = exp2 back into the place of S, as fp16.  Two and a half
//     instructions a score: packed fp32 pairs, and no search for the maximum (below).
//
// A key block's scale multiplies its columns of S in the same instruction that subtracts the maximum.  The value scale goes into
// the exponent, w = exp2(x - m + log2(scale / reference)), so that P V needs none; the row sum takes it out again, 16 columns
// at a time.  The reference is the first block's largest scale; O is rescaled where a block's largest leaves it by 2^6.  P is
// computed with the maximum of the blocks before; only where the weights of 16 keys sum to more than 2^14 (fp16 ends at 2^16)
// the block's maximum is looked for and P computed again.  P is rounded to fp16 (2^-11 of each weight; with many keys the roundings average out, and in
// the result they weigh as much as its own rounding).
//
// Shares, parts and their joining: kv8_attention.cuh, a CTA being a worker and a block of 128 keys a step.
#include <type_traits>

#include "kv8_attention.cuh"

LIGER_REGISTER_WAIT_BUDGET()

namespace liger {
namespace {

constexpr int kBlock = 128;         // keys of a block, rows of a half
constexpr int kItemRows = 256;
constexpr int kItemCost = 2;        // what it costs to begin a tile, in blocks
constexpr int kMinPlaces = 4;       // places that are worth a CTA
constexpr int kSoftmaxWarps = 8, kCodeWarps = 8, kQueryWarps = 3;
constexpr int kProductWarp = kSoftmaxWarps + kCodeWarps;
// Five warpgroups of 96 registers a thread at launch, 640 * 96 in all; 256 * 144 + 256 * 72 + 128 * 48 is as much.
constexpr int kThreads = 640;
constexpr int kSoftmaxRegs = 144, kCodeRegs = 72, kProductRegs = 48;
constexpr float kLargestSum = 16384.0f;
constexpr int kBox = 128 * 128;     // 128 rows x 64 fp16
constexpr int kSlots = 4;           // scales of blocks

template <int D>
struct Cfg {
  static constexpr int kTile = D / 64 * kBox;
  static constexpr int kScaleBytes = kSlots * (8 * 16 + 16);
  static constexpr int kSmem = 6 * kTile /* Q x2, K x2, V x2 */ + kScaleBytes + 256 + 1024;
  static constexpr int kPart = kItemRows * (D + 2);
};

// V as B operand: dims along the 128-byte rows, keys across them
__device__ __forceinline__ uint64_t make_v_desc(uint32_t smem_addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((lbo >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
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
// waits for all loads so far; names the registers so that nothing uses them before
__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
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

// ---- the share of a CTA, tile by tile; every role walks it by itself -----------------------------------------------------------
struct Tile {
  int n0, n1;  // blocks that the halves see
  __device__ __forceinline__ int blocks() const { return max(n0, n1); }
  __device__ __forceinline__ int places() const { return max(1, blocks()) + kItemCost; }
};
// keys that row r of an entry sees
__device__ __forceinline__ int limit_of(const Kv8AttnParams& p, const Entry& e, int r) {
  return p.causal ? min(e.len, max(0, e.len - e.n + r / p.group + 1)) : e.len;
}
__device__ __forceinline__ Tile tile_of(const Kv8AttnParams& p, const Entry& e, int rt) {
  const int rows = e.n * p.group, r0 = rt * kItemRows;
  Tile t;
  t.n0 = r0 < rows ? (limit_of(p, e, min(r0 + 127, rows - 1)) + kBlock - 1) / kBlock : 0;
  t.n1 = r0 + 128 < rows ? (limit_of(p, e, min(r0 + 255, rows - 1)) + kBlock - 1) / kBlock : 0;
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
    at = share_begin(sh.total, sh.used, blockIdx.x);
    end = share_begin(sh.total, sh.used, blockIdx.x + 1);
    b = sh.b[0];
    e = load_entry(p, b, false);
    const long long inside = at - sh.first[0], per = head_places(p, e);
    head = (int)(inside / per);
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
          ++b;
          e = load_entry(p, b, false);
        } while (e.n == 0);
      }
    }
    cut(p);
  }
  // blocks of half h in this share: [s0, stop(h))
  __device__ __forceinline__ int stop(int h) const { return max(s0, min(s1, h ? t.n1 : t.n0)); }
  __device__ __forceinline__ int stop() const { return max(stop(0), stop(1)); }
  __device__ __forceinline__ bool complete() const { return s0 == 0 && s1 == max(1, t.blocks()); }
};

template <int D, int TYPE>
__global__ void __launch_bounds__(kThreads, 1) kv8_attention_tc_kernel(const Kv8AttnParams p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;                 // [2]
  uint8_t* sK = sQ + 2 * C::kTile;    // [2]
  uint8_t* sV = sK + 2 * C::kTile;    // [2]
  float4* s_scale = reinterpret_cast<float4*>(sV + 2 * C::kTile);      // [slots][8]: key scale, log2 of value scale, its inverse, mask
  float4* s_ref = s_scale + kSlots * 8;                                // [slots]: reference, old reference / new one, not plain
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_ref + kSlots);
  uint64_t* k_full = bars + 2;     // [2]
  uint64_t* k_empty = bars + 4;    // [2]
  uint64_t* v_full = bars + 6;     // [2]
  uint64_t* v_empty = bars + 8;    // [2]
  uint64_t* sc_full = bars + 10;   // [4]
  uint64_t* s_full = bars + 14;    // [2] halves
  uint64_t* p_full = bars + 16;    // [2]
  uint64_t* o_full = bars + 18;    // [2]
  uint64_t* o_empty = bars + 20;   // [2]
  uint64_t* q_full = bars;         // [2]
  uint64_t* q_empty = bars + 22;   // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  __shared__ Kv8Shares<1> shares;
  __shared__ Walk walks[kThreads / 32];  // a warp's place in its share; in shared memory, since registers are short

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], kQueryWarps);
      mbar_init(&q_empty[i], 1);
      mbar_init(&k_full[i], kCodeWarps);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], kCodeWarps);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < kSlots; ++i) mbar_init(&sc_full[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kProductWarp) {
    tmem_alloc(tmem_slot, 512);  // S at columns 0 / 128, O at 256 / 384
    tmem_relinquish();
  }
  tc_fence_before();
  find_shares<kThreads>(p, kMinPlaces, [&](const Entry& x) { return (long long)p.c.kv_heads * head_places(p, x); }, shares);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int worker = blockIdx.x;
  Walk& w = walks[warp];
  if (lane == 0) w.start(p, shares);
  __syncwarp();
  auto advance = [&]() {
    __syncwarp();
    if (lane == 0) w.next(p);
    __syncwarp();
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
    if (!p.by_tile && cw == 0 && lane == 0) p.records[worker].x = -1;
    for (; w.valid && ok; advance()) {
      if (cw == 0 && lane == 0 && w.s0 == 0 && w.s1 > 0) {  // who begins a tile knows who ends it
        const bool complete = w.complete();
        const int tile = w.head * tiles_of(p, w.e) + w.rt;
        if (p.by_tile || !complete) {
          p.records[p.by_tile ? (size_t)w.b * p.tiles + tile : (size_t)worker] =
              complete ? make_int2(-1, 0) : make_int2(worker, share_of(shares.total, shares.used, w.tile0 + w.t.places() - 1));
          if (!p.by_tile) p.tile_of[worker] = make_int4(w.b, tile, 0, 0);
        }
      }
      const int stop = w.stop(), s0 = w.s0, len = w.e.len, head = w.head;
      if (stop <= s0) continue;
      const int* row_table = p.c.table + (size_t)w.e.slot * p.c.max_pages;
      // lane i: page of 16-key group i & 7 of a block, then its key scale (lanes 0 .. 7) or value scale (8 .. 15)
      auto page_at = [&](int j) {
        const int key = j * kBlock + (lane & 7) * 16;
        return lane < 16 && j < stop && key < len ? __ldg(row_table + (key >> p.c.page_shift)) : -1;
      };
      auto valid_page = [&](int page, int j) {
        if (page >= 0 && page < p.c.num_pages) return page;
        if (cw == 0 && lane < 8 && j < stop && j * kBlock + lane * 16 < len)
          report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAttention + 3, w.b, (unsigned)page);
        return -1;
      };
      auto scale_at = [&](int page, int j) {
        if (page < 0) return 0.0f;
        const int key = j * kBlock + (lane & 7) * 16;
        const size_t ph = (size_t)page * p.c.kv_heads + head;
        return __ldg((lane < 8 ? p.c.ks : p.c.vs) + (ph << (p.c.page_shift - p.c.block_shift)) + ((key & page_mask) >> p.c.block_shift));
      };
      auto load = [&](const uint8_t* base, int j, int pages, uint4 (&x)[kPass]) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          const int key = j * kBlock + i * kKeysPass + r_in;
          const int page = __shfl_sync(0xffffffffu, pages, (i * kKeysPass >> 4) + group_in);
          x[i] = make_uint4(0, 0, 0, 0);
          if (page >= 0 && key < len)
            x[i] = __ldg(reinterpret_cast<const uint4*>(base + ((((size_t)page * p.c.kv_heads + head) << p.c.page_shift) + (key & page_mask)) * D + c * 16));
        }
      };
      auto store = [&](uint8_t* tile, const uint4 (&x)[kPass]) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
          const int r = i * kKeysPass + r_in;
          uint8_t* row = tile + (c >> 2) * kBox + r * 128;
          const int idx = (c & 3) * 2;
          const uint32_t a = kv8_bias<TYPE>(x[i].x), b = kv8_bias<TYPE>(x[i].y), d = kv8_bias<TYPE>(x[i].z), e = kv8_bias<TYPE>(x[i].w);
          *reinterpret_cast<uint4*>(row + ((idx ^ (r & 7)) << 4)) =
              make_uint4(kv8_pair<TYPE, 0>(a), kv8_pair<TYPE, 1>(a), kv8_pair<TYPE, 0>(b), kv8_pair<TYPE, 1>(b));
          *reinterpret_cast<uint4*>(row + (((idx + 1) ^ (r & 7)) << 4)) =
              make_uint4(kv8_pair<TYPE, 0>(d), kv8_pair<TYPE, 1>(d), kv8_pair<TYPE, 0>(e), kv8_pair<TYPE, 1>(e));
        }
      };
      auto publish = [&](uint64_t* bar) {
        fence_proxy_async();  // the tile is read by the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      };

      // pages of block j + 1 are looked up when block j begins, its scales then, its codes when block j has been laid down
      uint4 xk[kPass], xv[kPass];
      int page_now = valid_page(page_at(s0), s0), page_next = page_at(s0 + 1);
      float scale_now = scale_at(page_now, s0);
      load(p.c.k, s0, page_now, xk);
      load(p.c.v, s0, page_now, xv);

      float ref = 0.0f;
      for (int j = s0; j < stop; ++j, ++g) {
        const uint32_t st = g & 1u, ph = (g >> 1) & 1u;
        page_next = valid_page(page_next, j + 1);
        const float scale_next = scale_at(page_next, j + 1);
        const int page_after = page_at(j + 2);
        if (!mbar_wait_bounded(&k_empty[st], ph ^ 1u, abort_flag)) { ok = false; break; }
        if (cw == 0) {
          // scales of the block's eight groups: lanes 0 .. 7
          const float mine = scale_now < INFINITY ? scale_now : NAN;
          const float vs = __shfl_sync(0xffffffffu, mine, (lane & 7) + 8);
          const bool use = lane < 8 && page_now >= 0 && vs > 0.0f;
          const float top = warp_max(use ? vs : 0.0f);
          float moved = 1.0f;
          if (ref == 0.0f) {
            ref = top;
          } else if (top > 0.0f && (top > ref * 64.0f || top < ref * 0.015625f)) {
            moved = ref / top;
            ref = top;
          }
          const float base = ref > 0.0f ? ref : 1.0f;
          if (lane < 8)
            s_scale[(g & 3u) * 8 + lane] = make_float4(page_now >= 0 ? mine * p.scale_log2 : 0.0f,
                                                       page_now < 0 ? -INFINITY : vs > 0.0f ? __log2f(vs / base) : vs == 0.0f ? 0.0f : NAN,
                                                       use ? base / vs : 1.0f, page_now < 0 ? -INFINITY : 0.0f);
          const bool odd = __any_sync(0xffffffffu, lane < 16 && mine != mine);
          if (lane == 0) s_ref[g & 3u] = make_float4(base, moved, odd ? 1.0f : 0.0f, 0.0f);
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[g & 3u]);
        }
        store(sK + st * C::kTile, xk);
        publish(&k_full[st]);
        load(p.c.k, j + 1, page_next, xk);
        if (!mbar_wait_bounded(&v_empty[st], ph ^ 1u, abort_flag)) { ok = false; break; }
        // values of zero scale are zeros whatever their codes are
        const unsigned zero = __ballot_sync(0xffffffffu, lane >= 8 && lane < 16 && scale_now == 0.0f) >> 8;
        if (zero) {
#pragma unroll
          for (int i = 0; i < kPass; ++i)
            if (zero >> ((i * kKeysPass >> 4) + group_in) & 1u) xv[i] = make_uint4(0, 0, 0, 0);
        }
        store(sV + st * C::kTile, xv);
        publish(&v_full[st]);
        load(p.c.v, j + 1, page_next, xv);
        page_now = page_next;
        scale_now = scale_next;
        page_next = page_after;
      }
    }
  } else if (warp >= kProductWarp) {
    // ===== products =====
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProductRegs));
    if (warp == kProductWarp && lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128);
      constexpr uint32_t idesc_o = make_idesc_f16(128, D) | (1u << 16);  // B with dims contiguous
      uint32_t g = 0, nq[2] = {0, 0}, np[2] = {0, 0}, no[2] = {0, 0};
      bool ok = true;
      for (; w.valid && ok; w.next(p)) {
        const int s0 = w.s0, stop = w.stop(), e0 = w.stop(0), e1 = w.stop(1);
        if (stop <= s0) continue;
        auto issue_s = [&](int h, int j, int end) {
          const uint32_t n = g + (uint32_t)(j - s0), st = n & 1u;
          if (j == s0) {
            if (!mbar_wait_bounded(&q_full[h], nq[h] & 1u, abort_flag)) { ok = false; return; }
            ++nq[h];
          }
          if (!mbar_wait_bounded(&k_full[st], (n >> 1) & 1u, abort_flag)) { ok = false; return; }
          tc_fence_after();
          const uint32_t qa = smem_u32(sQ + h * C::kTile), ka = smem_u32(sK + st * C::kTile);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t da = make_sw128_kmajor_desc(qa + (k >> 2) * kBox) + (uint64_t)((k & 3) * 2);
            const uint64_t db = make_sw128_kmajor_desc(ka + (k >> 2) * kBox) + (uint64_t)((k & 3) * 2);
            umma_f16(tmem + h * 128, da, db, idesc_s, k != 0 ? 1u : 0u);
          }
          umma_commit(&s_full[h]);
          if (j == end - 1) umma_commit(&q_empty[h]);
        };
        auto issue_o = [&](int h, int j, int end) {
          const uint32_t n = g + (uint32_t)(j - s0), st = n & 1u;
          if (!mbar_wait_bounded(&v_full[st], (n >> 1) & 1u, abort_flag)) { ok = false; return; }
          if (!mbar_wait_bounded(&p_full[h], np[h] & 1u, abort_flag)) { ok = false; return; }
          ++np[h];
          if (j == s0) {
            if (!mbar_wait_bounded(&o_empty[h], (no[h] & 1u) ^ 1u, abort_flag)) { ok = false; return; }
            ++no[h];
          }
          tc_fence_after();
          const uint32_t va = smem_u32(sV + st * C::kTile);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 keys each
            umma_f16_ts(tmem + 256 + h * 128, tmem + h * 128 + k * 8, make_v_desc(va + k * 2048, kBox, 1024), idesc_o, (j != s0 || k != 0) ? 1u : 0u);
          if (j == end - 1) umma_commit(&o_full[h]);
        };
        if (s0 < e0) issue_s(0, s0, e0);
        if (ok && s0 < e1) issue_s(1, s0, e1);
        if (!ok) break;
        umma_commit(&k_empty[g & 1u]);
        for (int j = s0; j < stop && ok; ++j) {
          if (j < e0) {
            issue_o(0, j, e0);
            if (ok && j + 1 < e0) issue_s(0, j + 1, e0);
          }
          if (ok && j < e1) {
            issue_o(1, j, e1);
            if (ok && j + 1 < e1) issue_s(1, j + 1, e1);
          }
          if (!ok) break;
          const uint32_t n = g + (uint32_t)(j - s0);
          umma_commit(&v_empty[n & 1u]);
          if (j + 1 < stop) umma_commit(&k_empty[(n + 1) & 1u]);
        }
        g += (uint32_t)(stop - s0);
      }
    } else if (warp > kProductWarp) {
      // ===== queries =====
      const int qt = threadIdx.x - (kProductWarp + 1) * 32;
      constexpr int kQChunks = D / 8;
      uint32_t nq[2] = {0, 0};
      bool ok = true;
      for (; w.valid && ok; advance()) {
        const int rows = w.e.n * p.group;
        const __half* base = p.q + (p.e.q_offsets ? (long long)w.e.row0 * p.q_token_stride : (long long)w.b * p.q_batch_stride) +
                             (long long)w.head * p.group * p.q_head_stride;
        for (int h = 0; h < 2 && ok; ++h) {
          if (w.stop(h) <= w.s0) continue;
          if (!mbar_wait_bounded(&q_empty[h], (nq[h] & 1u) ^ 1u, abort_flag)) { ok = false; break; }
          ++nq[h];
          const int r0 = w.rt * kItemRows + h * 128;
          for (int i = qt; i < 128 * kQChunks; i += kQueryWarps * 32) {
            const int rr = i / kQChunks, qc = i % kQChunks, r = r0 + rr;
            const uint32_t dst = smem_u32(sQ + h * C::kTile + (qc >> 3) * kBox + rr * 128 + (((qc & 7) ^ (rr & 7)) << 4));
            const __half* src = r < rows ? base + (long long)(r / p.group) * p.q_token_stride + (long long)(r % p.group) * p.q_head_stride + qc * 8 : p.q;
            const int bytes = r < rows ? 16 : 0;  // rows that are not there are zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[h]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ===== softmax and output: thread = row of half h =====
    const int h = warp >> 2, quad = warp & 3;
    const int r_tile = h * 128 + quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + h * 128 + lanes, o_addr = tmem + 256 + h * 128 + lanes;
    uint32_t g = 0, ns = 0, no = 0;
    bool ok = true;
    for (; w.valid && ok; advance()) {
      const int s0 = w.s0, stop = w.stop(h), all = w.stop();
      if (w.s1 == 0) continue;
      const int rows = w.e.n * p.group, r = w.rt * kItemRows + r_tile;
      const int limit = r < rows ? limit_of(p, w.e, r) : 0;
      // the first row of this warp that exists sees least
      const int r_low = w.rt * kItemRows + h * 128 + quad * 32;
      const int limit_low = r_low + 31 < rows ? limit_of(p, w.e, r_low) : 0;
      float m_ref = -INFINITY, l = 0.0f, ref = 1.0f;
      for (int j = s0; j < stop; ++j, ++ns) {
        const uint32_t slot = (g + (uint32_t)(j - s0)) & 3u;
        if (!mbar_wait_bounded(&sc_full[slot], ((g + (uint32_t)(j - s0)) >> 2) & 1u, abort_flag) ||
            !mbar_wait_bounded(&s_full[h], ns & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const float4* sc = s_scale + slot * 8;
        const float4 rf = s_ref[slot];
        ref = rf.x;
        const int cut = limit - j * kBlock;  // columns from here on are not seen
        // the same in the whole warp: nothing is hidden from a row, no page is missing, no scale is not finite
        const bool plain = limit_low - j * kBlock >= kBlock && rf.z == 0.0f;
        float m_try = m_ref, alpha = rf.y;
        uint32_t pk[64];
        float sum;
        bool large;
        auto weigh = [&](auto all_plain) {
          const float m_safe = m_try == -INFINITY ? 0.0f : m_try;
          sum = 0.0f;
          large = false;
          uint32_t v[2][16];
          tmem_ld_32x16(s_addr, v[0]);
#pragma unroll
          for (int gi = 0; gi < 8; ++gi) {
            tmem_ld_wait16(v[gi & 1]);
            if (gi < 7) tmem_ld_32x16(s_addr + (gi + 1) * 16, v[(gi + 1) & 1]);
            const uint32_t(&x)[16] = v[gi & 1];
            const float4 f = sc[gi];
            const float off = f.y - m_safe;
            float total;
            if constexpr (decltype(all_plain)::value) {
              const uint64_t f2 = pack2(f.x, f.x), off2 = pack2(off, off);
              uint64_t a = 0, b = 0;
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const float2 y0 = unpack2(fma2(pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), f2, off2));
                const float2 y1 = unpack2(fma2(pack2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), f2, off2));
                const float w0 = exp2_approx(y0.x), w1 = exp2_approx(y0.y), w2 = exp2_approx(y1.x), w3 = exp2_approx(y1.y);
                a = add2(a, pack2(w0, w1));
                b = add2(b, pack2(w2, w3));
                pk[gi * 8 + (i >> 1)] = pack_half2(w0, w1);
                pk[gi * 8 + (i >> 1) + 1] = pack_half2(w2, w3);
              }
              const float2 ab = unpack2(add2(a, b));
              total = ab.x + ab.y;
            } else {
              total = 0.0f;
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                float w0 = exp2_approx(fmaf(__uint_as_float(x[i]), f.x, off)), w1 = exp2_approx(fmaf(__uint_as_float(x[i + 1]), f.x, off));
                w0 = gi * 16 + i < cut ? w0 : 0.0f;
                w1 = gi * 16 + i + 1 < cut ? w1 : 0.0f;
                total += w0 + w1;
                pk[gi * 8 + (i >> 1)] = pack_half2(w0, w1);
              }
            }
            large |= total > kLargestSum;
            sum = fmaf(total, f.z, sum);
          }
        };
        // a row's first sight of keys, or weights that grew too large: its largest score
        bool seek = m_try == -INFINITY && cut > 0;
        for (;;) {
          if (__any_sync(0xffffffffu, seek)) {
            float mx = -INFINITY;
#pragma unroll 1
            for (int gi = 0; gi < 8; ++gi) {
              uint32_t v[16];
              tmem_ld_32x16(s_addr + gi * 16, v);
              tmem_ld_wait16(v);
              const float4 f = sc[gi];
              float a = -INFINITY;
#pragma unroll
              for (int i = 0; i < 16; ++i) a = gi * 16 + i < cut ? fmaxf(a, __uint_as_float(v[i])) : a;
              mx = fmaxf(mx, a == -INFINITY ? a : fmaf(a, f.x, f.w));
            }
            if (seek) m_try = fmaxf(m_try, mx);
          }
          if (plain) weigh(std::true_type{});
          else weigh(std::false_type{});
          if (!__any_sync(0xffffffffu, large)) break;
          seek = large;
        }
        if (m_try != m_ref) {
          alpha = m_ref == -INFINITY ? 0.0f : alpha * exp2_approx(m_ref - m_try);
          l *= m_ref == -INFINITY ? 0.0f : exp2_approx(m_ref - m_try);
          m_ref = m_try;
        }
        l += sum;
        if (j > s0 && __any_sync(0xffffffffu, alpha != 1.0f)) {  // the products so far are complete: S came after them
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t v[32];
            tmem_ld_32x32(o_addr + ch * 32, v);
            tmem_ld_wait_regs(v);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
            tmem_st_32x32(o_addr + ch * 32, v);
          }
        }
        // P in the place of S
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = pk[ch * 32 + i];
          tmem_st_32x32(s_addr + ch * 32, v);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[h]);
      }
      if (!ok) break;
      g += (uint32_t)(all > s0 ? all - s0 : 0);
      // the row's result, or its part
      const bool some = stop > s0, complete = w.complete();
      if (some) {
        if (!mbar_wait_bounded(&o_full[h], no & 1u, abort_flag)) { ok = false; break; }
        ++no;
        tc_fence_after();
      }
      const float inv = l == 0.0f ? 0.0f : ref / l;
      const int token = r / p.group;
      __half* out = p.out + (size_t)(w.e.row0 + token) * p.ldo + (size_t)(w.head * p.group + r % p.group) * D;
      float* part = p.parts + (size_t)(2 * worker + (w.first && s0 > 0 ? 0 : 1)) * C::kPart;
      if (!complete && r < rows) { part[r_tile] = m_ref; part[kItemRows + r_tile] = l; }
      part += 2 * kItemRows + (size_t)r_tile * D;
#pragma unroll 1
      for (int ch = 0; ch < D / 32; ++ch) {
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
        if (lane == 0) mbar_arrive(&o_empty[h]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProductWarp) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) report_failure(p.status, LIGER_DEV_TIMEOUT, 0x210u, blockIdx.x, 0);
}

template <int D, int TYPE>
int launch(const Kv8AttnParams& p, const Kv8AttnPlan& pl, cudaStream_t s) {
  LIGER_CUDA_TRY(cudaFuncSetAttribute(kv8_attention_tc_kernel<D, TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
  kv8_attention_tc_kernel<D, TYPE><<<pl.workers, kThreads, Cfg<D>::kSmem, s>>>(p);
  const int rc = check_launch("kv8_attention_tc_kernel");
  return rc != LIGER_OK ? rc : launch_join<D, kItemRows>(p, pl, s);
}

}  // namespace

int launch_kv8_attention_tc(const Kv8AttnParams& p, const Kv8AttnPlan& pl, int head_dim, int type, cudaStream_t s) {
  const DeviceInfo* dev = nullptr;
  const int rc = require_sm100(&dev);
  if (rc != LIGER_OK) return rc;
  if (head_dim == 128) return type == LIGER_KV8_INT8 ? launch<128, LIGER_KV8_INT8>(p, pl, s) : launch<128, LIGER_KV8_E4M3>(p, pl, s);
  return type == LIGER_KV8_INT8 ? launch<64, LIGER_KV8_INT8>(p, pl, s) : launch<64, LIGER_KV8_E4M3>(p, pl, s);
}

}  // namespace liger
