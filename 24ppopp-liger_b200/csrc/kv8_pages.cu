// Keeping the pages of the paged 8-bit cache: reserve, fork, free, copy, compact.
//
// Every operator but free and a small reserve is two launches.  A planning kernel of one CTA decides everything that depends on order (who gets
// which page), with prefix sums over the entries and over the pages' reference counts, and leaves a list of page moves in the
// workspace.  A second kernel over the whole GPU then carries it out: the entries' table rows and the bytes of the moved
// pages, which are what costs time (two launches, no trip to the host).  Which page goes where never hangs on timing:
// free pages are handed out lowest number first and entries are served in their order.
#include "kv8.cuh"

namespace liger {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kMovePiece = kMoveThreads * 8 * 16;
constexpr int kMostEntries = 1 << 28;  // of a call: entries times 8 warps stay within 32 bits
constexpr int kNobody = 0x7fffffff;
constexpr int kOwnersShared = 8192;   // slots or pages up to which the owners of a call's numbers are kept in shared memory
constexpr int kFreeShared = 2048;     // free pages handed out that are kept there
constexpr int kLook = 8;              // reference counts a thread looks at in a round

struct PagesParams {
  uint8_t *k, *v;
  float *ks, *vs;
  int *table, *count, *refs;
  int layers, num_pages, slots, max_pages, page_size;
  size_t page_codes;   // bytes of one page's codes in one layer
  int page_scales;     // scales of one page in one layer
  // the call
  const int *src, *dst, *lens;
  int n;
  int *done, *live, *moved_to;
  // the workspace
  int* n_moves;        // [16]
  int *from, *to;      // [moves]
  int* owner;          // [max(num_pages, slots)]
  int* free_list;      // [num_pages]
  int *first, *many;   // [n]: where an entry's new pages begin in free_list, and how many (-1: refused)
  DeviceStatus* status;
};

struct Workspace {
  size_t moves, owners, bytes;
};
Workspace workspace_of(const liger_kv8_cache* c, int n) {
  Workspace w;
  w.moves = (size_t)(c->num_pages > n ? c->num_pages : n);
  w.owners = (size_t)(c->num_pages > c->slots ? c->num_pages : c->slots);
  w.bytes = (16 + 2 * w.moves + w.owners + (size_t)c->num_pages + 2 * (size_t)n) * sizeof(int);
  w.bytes = (w.bytes + 15) & ~(size_t)15;
  return w;
}

// Exclusive prefix sum over the CTA's 1024 threads; `total` receives the sum.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T& total, T* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    T s = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    s_warp[lane] = s;
  }
  __syncthreads();
  const T before = warp ? s_warp[warp - 1] : 0;
  total = s_warp[31];
  __syncthreads();
  return before + incl - v;
}

// What a planning CTA keeps in shared memory; the same arrays lie in the workspace where they do not fit.
struct PlanShared {
  int warp[32];
  long long wide[32];
  int owner[kOwnersShared];
  int free_list[kFreeShared];
};

// Marks the first entry that names each number of `named` inside [0, limit).
__device__ __forceinline__ void mark_owners(const int* named, int n, int limit, int* owner) {
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int x = named[i];
    if (x >= 0 && x < limit) owner[x] = kNobody;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int x = named[i];
    if (x >= 0 && x < limit) atomicMin(owner + x, i);
  }
  __syncthreads();
}

// Which of the pages that a thread looks at in a round are free, bit by bit.
__device__ __forceinline__ unsigned look_at_refs(const PagesParams& p, int base) {
  const int at = base + (int)threadIdx.x * kLook;
  unsigned free = 0;
#pragma unroll
  for (int i = 0; i < kLook; ++i) free |= (unsigned)(at + i < p.num_pages && p.refs[at + i] == 0) << i;
  return free;
}

// The planning kernels take one trip to memory after the other (entries, counts, reference counts, table; 8 us with cold caches for
// 256 entries and 6000 pages): what can be known early is asked for early.
__device__ __forceinline__ void prefetch(const void* at) { asm volatile("prefetch.global.L1 [%0];" ::"l"(at)); }

// The first `wanted` free pages (all, if there are fewer), lowest number first, into the workspace and, those that fit, into
// shared memory; returns how many.  `free`: of the first round.
__device__ int list_free(const PagesParams& p, int wanted, unsigned free, PlanShared& s) {
  int found = 0;
  for (int base = 0; base < p.num_pages && found < wanted; base += kPlanThreads * kLook) {
    const int at = base + (int)threadIdx.x * kLook;
    if (base > 0) free = look_at_refs(p, base);
    int total, rank = found + block_prefix(__popc(free), total, s.warp);
#pragma unroll
    for (int i = 0; i < kLook; ++i)
      if (free >> i & 1u) {
        p.free_list[rank] = at + i;
        if (rank < kFreeShared) s.free_list[rank] = at + i;
        ++rank;
      }
    found += total;
  }
  __syncthreads();
  return found;
}

// Hands out pages.  `want(i)` gives how many entry i wants (-1: refused already), `got(i, first, n)` is told where its pages begin in
// the list and how many they are (-1: refused).  Entries whose pages end behind the last free one are refused.  Returns the
// number of pages handed out.  Up to 1024 entries stay in their threads' registers.
template <typename Want, typename Got>
__device__ int hand_out(const PagesParams& p, PlanShared& s, unsigned free, Want want, Got got) {
  const long long most = (long long)p.num_pages + 1;  // more than there are: refused, whatever it is exactly
  long long ends = 0;
  int first = 0, many = -1;
  for (int base = 0; base < p.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    many = i < p.n ? want(i) : -1;
    long long total;
    first = (int)min(ends + block_prefix<long long>(max(0, many), total, s.wide), most);
    ends += total;
    if (p.n > kPlanThreads && i < p.n) {
      p.first[i] = first;
      p.many[i] = many;
    }
  }
  const int found = list_free(p, (int)min(ends, (long long)p.num_pages), free, s);
  int given = 0;
  for (int base = 0; base < p.n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    if (p.n > kPlanThreads && i < p.n) {
      first = p.first[i];
      many = p.many[i];
    }
    if (i >= p.n) many = -1;
    if (many > 0 && many > found - first) many = -1;
    int total;
    block_prefix(max(0, many), total, s.warp);
    given += total;
    if (i < p.n) {
      if (p.done) p.done[i] = many >= 0;
      got(i, first, many);
    }
  }
  return given;
}

__device__ __forceinline__ int* owners_of(const PagesParams& p, PlanShared& s, int limit) { return limit <= kOwnersShared ? s.owner : p.owner; }
__device__ __forceinline__ int free_page(const PagesParams& p, const PlanShared& s, int i) { return i < kFreeShared ? s.free_list[i] : p.free_list[i]; }

// here = 1: the entries' table rows are written by this CTA, else left to kv8_reserve_kernel
__global__ void __launch_bounds__(kPlanThreads) kv8_reserve_plan_kernel(const PagesParams p, int here) {
  extern __shared__ __align__(16) uint8_t smem_plan[];
  PlanShared& s = *reinterpret_cast<PlanShared*>(smem_plan);
  wait_for_stream();
  const unsigned free = look_at_refs(p, 0);
  if ((int)threadIdx.x < p.n) {
    const int slot = p.dst[threadIdx.x];
    if (slot >= 0 && slot < p.slots) prefetch(p.count + slot);
    prefetch(p.lens + threadIdx.x);
  }
  int* owner = owners_of(p, s, p.slots);
  mark_owners(p.dst, p.n, p.slots, owner);
  hand_out(
      p, s, free,
      [&](int i) {
        const int slot = p.dst[i], len = p.lens[i];
        if (slot < 0 || slot >= p.slots || len < 0) {
          report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages, i, (unsigned)slot);
          return -1;
        }
        const int need = len / p.page_size + (len % p.page_size != 0);
        return owner[slot] == i && need <= p.max_pages ? max(0, need - max(0, p.count[slot])) : -1;
      },
      [&](int i, int first, int many) {
        if (here && many > 0) {
          const int slot = p.dst[i], had = max(0, p.count[slot]);
          int* row = p.table + (size_t)slot * p.max_pages + had;
          for (int j = 0; j < many; ++j) {
            const int page = free_page(p, s, first + j);
            row[j] = page;
            p.refs[page] = 1;
          }
          p.count[slot] = had + many;
        } else if (!here) {
          p.first[i] = first;
          p.many[i] = many;
        }
      });
}

__global__ void __launch_bounds__(kPlanThreads) kv8_fork_plan_kernel(const PagesParams p) {
  extern __shared__ __align__(16) uint8_t smem_plan[];
  PlanShared& s = *reinterpret_cast<PlanShared*>(smem_plan);
  wait_for_stream();
  const unsigned free = look_at_refs(p, 0);
  if ((int)threadIdx.x < p.n) {
    const int src = p.src[threadIdx.x], dst = p.dst[threadIdx.x], part = p.lens[threadIdx.x] / p.page_size;
    if (dst >= 0 && dst < p.slots) prefetch(p.count + dst);
    if (src >= 0 && src < p.slots) {
      prefetch(p.count + src);
      if (part >= 0 && part < p.max_pages) prefetch(p.table + (size_t)src * p.max_pages + part);
    }
  }
  int* owner = owners_of(p, s, p.slots);
  mark_owners(p.dst, p.n, p.slots, owner);
  const int given = hand_out(
      p, s, free,
      [&](int i) {
        const int src = p.src[i], dst = p.dst[i], len = p.lens[i];
        if (src < 0 || src >= p.slots || dst < 0 || dst >= p.slots || len < 0) {
          report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages + 1, i, (unsigned)dst);
          return -1;
        }
        const int full = len / p.page_size, part = len % p.page_size != 0;
        return owner[dst] == i && src != dst && p.count[dst] == 0 && full + part <= min(p.count[src], p.max_pages) ? part : -1;
      },
      [&](int i, int first, int many) {
        p.first[i] = first;
        p.many[i] = many;
        if (many > 0) {
          const int to = free_page(p, s, first);
          int from = p.table[(size_t)p.src[i] * p.max_pages + p.lens[i] / p.page_size];
          if (from < 0 || from >= p.num_pages) {
            report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages + 3, i, (unsigned)from);
            from = to;  // nothing to copy
          }
          p.from[first] = from;
          p.to[first] = to;
        }
      });
  if (threadIdx.x == 0) *p.n_moves = given;
}

__global__ void __launch_bounds__(kPlanThreads) kv8_copy_plan_kernel(const PagesParams p) {
  extern __shared__ __align__(16) uint8_t smem_plan[];
  PlanShared& sh = *reinterpret_cast<PlanShared*>(smem_plan);
  __shared__ int s_moves;
  wait_for_stream();
  if (threadIdx.x == 0) s_moves = 0;
  int* owner = owners_of(p, sh, p.num_pages);
  for (int i = threadIdx.x; i < p.n; i += kPlanThreads) {
    const int s = p.src[i];
    if (s >= 0 && s < p.num_pages) owner[s] = kNobody;
  }
  mark_owners(p.dst, p.n, p.num_pages, owner);
  for (int i = threadIdx.x; i < p.n; i += kPlanThreads) {
    const int s = p.src[i], d = p.dst[i];
    bool ok = false;
    if (s < 0 || s >= p.num_pages || d < 0 || d >= p.num_pages) {
      report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages + 2, i, (unsigned)d);
    } else {
      ok = owner[d] == i && (s == d || owner[s] == kNobody);
      if (ok && s != d) {
        const int m = atomicAdd(&s_moves, 1);  // the order of the moves does not matter: their targets differ
        p.from[m] = s;
        p.to[m] = d;
      }
    }
    if (p.done) p.done[i] = ok;
  }
  __syncthreads();
  if (threadIdx.x == 0) *p.n_moves = s_moves;
}

__global__ void __launch_bounds__(kPlanThreads) kv8_compact_plan_kernel(const PagesParams p) {
  __shared__ int s_warp[32];
  wait_for_stream();
  int mine = 0, live, total;
  for (int i = threadIdx.x; i < p.num_pages; i += kPlanThreads) mine += p.refs[i] != 0;
  block_prefix(mine, live, s_warp);
  // holes before `live` and pages in use behind it are equally many; the i-th of one goes to the i-th of the other
  int holes = 0, late = 0;
  for (int base = 0; base < p.num_pages; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    const bool used = i < p.num_pages && p.refs[i] != 0;
    const bool hole = i < live && !used, moves = i >= live && used;
    const int r = block_prefix(hole || moves ? (hole ? 1 : 0x10000) : 0, total, s_warp);  // 16 bits each: at most 1024 of a round
    if (hole) p.to[holes + (r & 0xffff)] = i;
    if (moves) p.from[late + (r >> 16)] = i;
    if (i < p.num_pages) p.moved_to[i] = used ? i : -1;
    holes += total & 0xffff;
    late += total >> 16;
  }
  __syncthreads();
  for (int m = threadIdx.x; m < late; m += kPlanThreads) {
    const int a = p.from[m], b = p.to[m];
    p.moved_to[a] = b;
    p.refs[b] = p.refs[a];
    p.refs[a] = 0;
  }
  if (threadIdx.x == 0) {
    *p.n_moves = late;
    if (p.live) *p.live = live;
  }
}

// Copies the planned pages, 32 KB of one page, layer and array at a time: eight loads a thread under way, five CTAs an SM (fork: four) at a time (of
// the grid's eight; registers).  600 pages of 786 KB (4 layers, 12 heads of 128, 64 tokens): 163 us, 5.8 TB/s of reads and writes, 89 % of the
// copy rate; 16 KB at a time cost 4 us more.
__device__ __forceinline__ void move_pages(const PagesParams& p) {
  constexpr int kU = kMovePiece / (kMoveThreads * 16), kPiece = kMovePiece;
  const int moves = *p.n_moves;
  const long long pieces = (long long)((p.page_codes + kPiece - 1) / kPiece);
  const long long per_page = 2 * pieces, all = (long long)moves * p.layers * per_page;
  for (long long w = blockIdx.x; w < all; w += gridDim.x) {
    const long long which = w / per_page;
    const int rest = (int)(w % per_page);
    const int layer = (int)(which % p.layers), m = (int)(which / p.layers);
    const bool is_v = rest >= pieces;
    const size_t at = (size_t)(is_v ? rest - pieces : rest) * kPiece;
    const size_t from = (size_t)layer * p.num_pages + p.from[m], to = (size_t)layer * p.num_pages + p.to[m];
    uint8_t* codes = is_v ? p.v : p.k;
    const uint4* s = reinterpret_cast<const uint4*>(codes + from * p.page_codes + at);
    uint4* d = reinterpret_cast<uint4*>(codes + to * p.page_codes + at);
    const int left = (int)((p.page_codes - at < (size_t)kPiece ? p.page_codes - at : (size_t)kPiece) / 16);
    uint4 x[kU];
#pragma unroll
    for (int i = 0; i < kU; ++i)
      if ((int)threadIdx.x + i * kMoveThreads < left) x[i] = __ldcs(s + threadIdx.x + i * kMoveThreads);
#pragma unroll
    for (int i = 0; i < kU; ++i)
      if ((int)threadIdx.x + i * kMoveThreads < left) __stcs(d + threadIdx.x + i * kMoveThreads, x[i]);
    if (at == 0) {
      float* sc = is_v ? p.vs : p.ks;
      for (int i = threadIdx.x; i < p.page_scales; i += kMoveThreads) sc[to * p.page_scales + i] = sc[from * p.page_scales + i];
    }
  }
}

__global__ void __launch_bounds__(kMoveThreads) kv8_move_kernel(const PagesParams p) {
  wait_for_stream();
  move_pages(p);
}

__global__ void __launch_bounds__(kMoveThreads) kv8_fork_kernel(const PagesParams p) {
  wait_for_stream();
  const int lane = threadIdx.x & 31;
  for (int i = (blockIdx.x * kMoveThreads + threadIdx.x) >> 5; i < p.n; i += gridDim.x * kMoveThreads / 32) {
    if (p.many[i] < 0) continue;
    const int full = p.lens[i] / p.page_size, part = p.many[i];
    const int* src = p.table + (size_t)p.src[i] * p.max_pages;
    int* dst = p.table + (size_t)p.dst[i] * p.max_pages;
    for (int j = lane; j < full; j += 32) {
      const int page = src[j];
      dst[j] = page;
      if (page >= 0 && page < p.num_pages) atomicAdd(p.refs + page, 1);
      else report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages + 3, i, (unsigned)page);
    }
    if (lane == 0) {
      if (part) {
        const int page = p.free_list[p.first[i]];
        dst[full] = page;
        p.refs[page] = 1;
      }
      p.count[p.dst[i]] = full + part;
    }
  }
  move_pages(p);
}

__global__ void __launch_bounds__(kMoveThreads) kv8_reserve_kernel(const PagesParams p) {
  wait_for_stream();
  const int lane = threadIdx.x & 31;
  for (int i = (blockIdx.x * kMoveThreads + threadIdx.x) >> 5; i < p.n; i += gridDim.x * kMoveThreads / 32) {
    const int more = p.many[i];
    if (more <= 0) continue;
    const int slot = p.dst[i], had = max(0, p.count[slot]);
    for (int j = lane; j < more; j += 32) {
      const int page = p.free_list[p.first[i] + j];
      p.table[(size_t)slot * p.max_pages + had + j] = page;
      p.refs[page] = 1;
    }
    __syncwarp();
    if (lane == 0) p.count[slot] = had + more;
  }
}

// One warp per entry.  Whoever takes the count frees the slot, so a slot that is named twice is freed once.
__global__ void __launch_bounds__(kMoveThreads) kv8_free_kernel(const PagesParams p) {
  wait_for_stream();
  const int lane = threadIdx.x & 31;
  const int i = (int)((blockIdx.x * (size_t)kMoveThreads + threadIdx.x) >> 5);
  if (i >= p.n) return;
  const int slot = p.dst[i];
  if (slot < 0 || slot >= p.slots) {
    if (lane == 0) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages + 4, i, (unsigned)slot);
    return;
  }
  int held = 0;
  if (lane == 0) held = atomicExch(p.count + slot, 0);
  held = min(__shfl_sync(0xffffffffu, held, 0), p.max_pages);
  int* row = p.table + (size_t)slot * p.max_pages;
  for (int j = lane; j < held; j += 32) {
    const int page = row[j];
    row[j] = -1;
    if (page < 0 || page >= p.num_pages || atomicSub(p.refs + page, 1) <= 0) {
      if (page >= 0 && page < p.num_pages) atomicAdd(p.refs + page, 1);
      report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtPages + 5, i, (unsigned)page);
    }
  }
}

__global__ void __launch_bounds__(kMoveThreads) kv8_compact_kernel(const PagesParams p) {
  wait_for_stream();
  const size_t entries = (size_t)p.slots * p.max_pages;
  for (size_t i = blockIdx.x * (size_t)kMoveThreads + threadIdx.x; i < entries; i += (size_t)gridDim.x * kMoveThreads) {
    const int page = p.table[i];
    if (page >= 0 && page < p.num_pages) p.table[i] = p.moved_to[page];
  }
  move_pages(p);
}

int check_n(const char* what, int n) {
  if (n < 0) return set_error(LIGER_ERR_INVALID, "%s: n must not be negative", what);
  if (n > kMostEntries) return set_error(LIGER_ERR_UNSUPPORTED, "%s: n <= %d", what, kMostEntries);
  return LIGER_OK;
}

int pages_params(const char* what, const liger_kv8_cache* c, int n, bool state, void* scratch, size_t scratch_bytes, PagesParams* p,
                 const DeviceInfo** dev) {
  int rc = kv8_check(what, c, -1);
  if (rc != LIGER_OK) return rc;
  if (state && (!c->page_count || !c->page_refs)) return set_error(LIGER_ERR_INVALID, "%s: page_count and page_refs are needed", what);
  if ((rc = check_n(what, n)) != LIGER_OK) return rc;
  const Workspace w = workspace_of(c, n);
  if (!scratch || ((uintptr_t)scratch & 15u)) return set_error(LIGER_ERR_INVALID, "%s: scratch must be a 16-byte aligned pointer", what);
  if (scratch_bytes < w.bytes)
    return set_error(LIGER_ERR_TOO_LARGE, "%s: scratch has %zu bytes, %zu are needed", what, scratch_bytes, w.bytes);
  *dev = current_device();
  if (!*dev) return LIGER_ERR_CUDA;
  *p = PagesParams{};
  p->k = (uint8_t*)c->k_pages;
  p->v = (uint8_t*)c->v_pages;
  p->ks = c->k_scales;
  p->vs = c->v_scales;
  p->table = c->page_table;
  p->count = c->page_count;
  p->refs = c->page_refs;
  p->layers = c->layers;
  p->num_pages = c->num_pages;
  p->slots = c->slots;
  p->max_pages = c->max_pages;
  p->page_size = c->page_size;
  p->page_codes = (size_t)c->kv_heads * c->page_size * c->head_dim;
  p->page_scales = c->kv_heads * (c->page_size / c->scale_block);
  p->n = n;
  p->status = (*dev)->status_dev;
  int* s = (int*)scratch;
  p->n_moves = s;
  s += 16;
  p->from = s;
  s += w.moves;
  p->to = s;
  s += w.moves;
  p->owner = s;
  s += w.owners;
  p->free_list = s;
  s += c->num_pages;
  p->first = s;
  p->many = s + n;
  return LIGER_OK;
}

int check_ints(const char* what, const int* a, const int* b, const int* c) {
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3u) return set_error(LIGER_ERR_INVALID, "%s: arrays must be 4-byte aligned", what);
  return LIGER_OK;
}

// as many CTAs as there can be pieces to move, at most eight an SM
unsigned move_grid(const DeviceInfo* dev, const PagesParams& p, long long moves) {
  const long long pieces = (moves < 1 ? 1 : moves) * p.layers * 2 * (long long)((p.page_codes + kMovePiece - 1) / kMovePiece);
  return (unsigned)(pieces < (long long)dev->sm_count * 8 ? pieces : (long long)dev->sm_count * 8);
}

}  // namespace
}  // namespace liger

using namespace liger;

extern "C" size_t liger_kv8_pages_scratch_bytes(const liger_kv8_cache* cache, int n) {
  if (!cache || cache->num_pages <= 0 || cache->slots <= 0 || n < 0 || n > kMostEntries) return 0;
  return workspace_of(cache, n).bytes;
}

extern "C" int liger_kv8_reserve(const liger_kv8_cache* cache, const int* slots, const int* lens, int n, int* done, void* scratch,
                                 size_t scratch_bytes, void* stream) {
  PagesParams p;
  const DeviceInfo* dev = nullptr;
  int rc = pages_params("kv8_reserve", cache, n, true, scratch, scratch_bytes, &p, &dev);
  if (rc != LIGER_OK || n == 0) return rc;
  if (!slots || !lens) return set_error(LIGER_ERR_INVALID, "kv8_reserve: slots or lens is NULL");
  if ((rc = check_ints("kv8_reserve", slots, lens, done)) != LIGER_OK) return rc;
  p.dst = slots;
  p.lens = lens;
  p.done = done;
  // few pages at most: the planning CTA writes them down itself (a second launch costs about 3 us; a thread writes a page in
  // about 20 ns)
  const int here = n <= kPlanThreads && cache->max_pages <= 256;
  rc = launch_early("kv8_reserve_plan_kernel", kv8_reserve_plan_kernel, 1, kPlanThreads, sizeof(PlanShared), (cudaStream_t)stream, p, here);
  if (rc != LIGER_OK || here) return rc;
  return launch_early("kv8_reserve_kernel", kv8_reserve_kernel, (unsigned)dev->sm_count, kMoveThreads, 0, (cudaStream_t)stream, p);
}

extern "C" int liger_kv8_fork(const liger_kv8_cache* cache, const int* src, const int* dst, const int* lens, int n, int* done,
                              void* scratch, size_t scratch_bytes, void* stream) {
  PagesParams p;
  const DeviceInfo* dev = nullptr;
  int rc = pages_params("kv8_fork", cache, n, true, scratch, scratch_bytes, &p, &dev);
  if (rc != LIGER_OK || n == 0) return rc;
  if (!src || !dst || !lens) return set_error(LIGER_ERR_INVALID, "kv8_fork: src, dst or lens is NULL");
  if ((rc = check_ints("kv8_fork", src, dst, lens)) != LIGER_OK || (rc = check_ints("kv8_fork", done, nullptr, nullptr)) != LIGER_OK) return rc;
  p.src = src;
  p.dst = dst;
  p.lens = lens;
  p.done = done;
  if ((rc = launch_early("kv8_fork_plan_kernel", kv8_fork_plan_kernel, 1, kPlanThreads, sizeof(PlanShared), (cudaStream_t)stream, p)) != LIGER_OK) return rc;
  return launch_early("kv8_fork_kernel", kv8_fork_kernel, move_grid(dev, p, n), kMoveThreads, 0, (cudaStream_t)stream, p);
}

extern "C" int liger_kv8_free(const liger_kv8_cache* cache, const int* slots, int n, void* stream) {
  int rc = kv8_check("kv8_free", cache, -1);
  if (rc != LIGER_OK) return rc;
  if (!cache->page_count || !cache->page_refs) return set_error(LIGER_ERR_INVALID, "kv8_free: page_count and page_refs are needed");
  if ((rc = check_n("kv8_free", n)) != LIGER_OK || n == 0) return rc;
  if (!slots) return set_error(LIGER_ERR_INVALID, "kv8_free: slots is NULL");
  if ((rc = check_ints("kv8_free", slots, nullptr, nullptr)) != LIGER_OK) return rc;
  const DeviceInfo* dev = current_device();
  if (!dev) return LIGER_ERR_CUDA;
  PagesParams p{};
  p.table = cache->page_table;
  p.count = cache->page_count;
  p.refs = cache->page_refs;
  p.num_pages = cache->num_pages;
  p.slots = cache->slots;
  p.max_pages = cache->max_pages;
  p.dst = slots;
  p.n = n;
  p.status = dev->status_dev;
  const unsigned grid = (unsigned)(((size_t)n * 32 + kMoveThreads - 1) / kMoveThreads);
  return launch_early("kv8_free_kernel", kv8_free_kernel, grid, kMoveThreads, 0, (cudaStream_t)stream, p);
}

extern "C" int liger_kv8_copy(const liger_kv8_cache* cache, const int* src, const int* dst, int n, int* done, void* scratch,
                              size_t scratch_bytes, void* stream) {
  PagesParams p;
  const DeviceInfo* dev = nullptr;
  int rc = pages_params("kv8_copy", cache, n, false, scratch, scratch_bytes, &p, &dev);
  if (rc != LIGER_OK || n == 0) return rc;
  if (!src || !dst) return set_error(LIGER_ERR_INVALID, "kv8_copy: src or dst is NULL");
  if ((rc = check_ints("kv8_copy", src, dst, done)) != LIGER_OK) return rc;
  p.src = src;
  p.dst = dst;
  p.done = done;
  if ((rc = launch_early("kv8_copy_plan_kernel", kv8_copy_plan_kernel, 1, kPlanThreads, sizeof(PlanShared), (cudaStream_t)stream, p)) != LIGER_OK) return rc;
  return launch_early("kv8_move_kernel", kv8_move_kernel, move_grid(dev, p, n), kMoveThreads, 0, (cudaStream_t)stream, p);
}

extern "C" int liger_kv8_compact(const liger_kv8_cache* cache, int* live, int* moved_to, void* scratch, size_t scratch_bytes,
                                 void* stream) {
  PagesParams p;
  const DeviceInfo* dev = nullptr;
  int rc = pages_params("kv8_compact", cache, 0, true, scratch, scratch_bytes, &p, &dev);
  if (rc != LIGER_OK) return rc;
  if ((rc = check_ints("kv8_compact", live, moved_to, nullptr)) != LIGER_OK) return rc;
  p.live = live;
  p.moved_to = moved_to ? moved_to : p.owner;
  if ((rc = launch_early("kv8_compact_plan_kernel", kv8_compact_plan_kernel, 1, kPlanThreads, 0, (cudaStream_t)stream, p)) != LIGER_OK) return rc;
  return launch_early("kv8_compact_kernel", kv8_compact_kernel, move_grid(dev, p, cache->num_pages), kMoveThreads, 0, (cudaStream_t)stream, p);
}
