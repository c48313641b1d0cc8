// Writing new keys and values into the paged 8-bit cache (liger_kv8_append), and the argument checks of its operators.
//
// A unit of work is one block of `scale_block` tokens of one head, keys or values.  Its threads hold all of the block's new
// values in registers (64 per thread), so that the values are read once: the largest magnitude is found with fp16
// maxima that keep a NaN (and between lanes with integer maxima of the bit patterns, in which a NaN is above infinity), then the
// codes are rounded and written.  A new value times the reciprocal is at most the largest code * (1 + 2^-22), so it rounds to
// a code without a bound.  The codes that a block already holds are only read
// when its scale grows.
#include "kv8.cuh"

namespace liger {

int kv8_check(const char* what, const liger_kv8_cache* c, int layer) {
  if (!c) return set_error(LIGER_ERR_INVALID, "%s: cache is NULL", what);
  if (!c->k_pages || !c->v_pages || !c->k_scales || !c->v_scales || !c->page_table)
    return set_error(LIGER_ERR_INVALID, "%s: a pointer of the cache is NULL", what);
  if (((uintptr_t)c->k_pages | (uintptr_t)c->v_pages) & 15u)
    return set_error(LIGER_ERR_INVALID, "%s: k_pages / v_pages must be 16-byte aligned", what);
  if (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales | (uintptr_t)c->page_table | (uintptr_t)c->page_count | (uintptr_t)c->page_refs) & 3u)
    return set_error(LIGER_ERR_INVALID, "%s: scales and tables must be 4-byte aligned", what);
  if (c->layers <= 0 || c->num_pages <= 0 || c->kv_heads <= 0 || c->slots <= 0 || c->max_pages <= 0)
    return set_error(LIGER_ERR_INVALID, "%s: layers, num_pages, kv_heads, slots and max_pages must be positive", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(LIGER_ERR_UNSUPPORTED, "%s: head_dim %d (64 and 128 are implemented)", what, c->head_dim);
  if (c->type != LIGER_KV8_INT8 && c->type != LIGER_KV8_E4M3) return set_error(LIGER_ERR_INVALID, "%s: type %d", what, c->type);
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return set_error(LIGER_ERR_UNSUPPORTED, "%s: page_size %d (powers of two from 16 to 256 are implemented)", what, c->page_size);
  if (c->scale_block < 16 || c->scale_block > 128 || c->scale_block > c->page_size || (c->scale_block & (c->scale_block - 1)))
    return set_error(LIGER_ERR_UNSUPPORTED, "%s: scale_block %d (powers of two from 16 to 128, at most page_size)", what, c->scale_block);
  if (c->num_pages > (1 << 30) || c->slots > (1 << 30)) return set_error(LIGER_ERR_UNSUPPORTED, "%s: num_pages and slots <= 2^30", what);
  if (c->kv_heads > 65535 || (long long)c->max_pages * c->page_size > (1ll << 30))
    return set_error(LIGER_ERR_UNSUPPORTED, "%s: kv_heads <= 65535, max_pages * page_size <= 2^30", what);
  if (layer >= c->layers) return set_error(LIGER_ERR_INVALID, "%s: layer %d of %d", what, layer, c->layers);
  return LIGER_OK;
}

static int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

Kv8Layer kv8_layer(const liger_kv8_cache* c, int layer) {
  const size_t blocks = (size_t)c->num_pages * c->kv_heads * (c->page_size / c->scale_block);
  const size_t codes = (size_t)c->num_pages * c->kv_heads * c->page_size * c->head_dim;
  Kv8Layer l;
  l.k = (uint8_t*)c->k_pages + codes * layer;
  l.v = (uint8_t*)c->v_pages + codes * layer;
  l.ks = c->k_scales + blocks * layer;
  l.vs = c->v_scales + blocks * layer;
  l.table = c->page_table;
  l.num_pages = c->num_pages;
  l.kv_heads = c->kv_heads;
  l.page_shift = log2_of(c->page_size);
  l.block_shift = log2_of(c->scale_block);
  l.slots = c->slots;
  l.max_pages = c->max_pages;
  return l;
}

int kv8_check_tokens(const char* what, const int* q_offsets, int batch, int q_len, int total_tokens, long long batch_stride,
                     long long token_stride, long long head_stride) {
  if (batch <= 0 || q_len <= 0) return set_error(LIGER_ERR_INVALID, "%s: batch and q_len must be positive", what);
  if (batch > 65535 || q_len > (1 << 29)) return set_error(LIGER_ERR_UNSUPPORTED, "%s: batch <= 65535, q_len <= 2^29", what);
  if (q_offsets ? total_tokens < 0 : (long long)batch * q_len > 0x7fffffffll)
    return set_error(LIGER_ERR_INVALID, "%s: the number of tokens must be between 0 and 2^31 - 1", what);
  if ((q_offsets == nullptr && batch_stride % 8) || token_stride % 8 || head_stride % 8)
    return set_error(LIGER_ERR_INVALID, "%s: strides must be multiples of 8 elements", what);
  if ((q_offsets == nullptr && batch_stride < 0) || token_stride < 0 || head_stride < 0)
    return set_error(LIGER_ERR_INVALID, "%s: strides must not be negative", what);
  if ((uintptr_t)q_offsets & 3u) return set_error(LIGER_ERR_INVALID, "%s: q_offsets must be 4-byte aligned", what);
  return LIGER_OK;
}

namespace {

constexpr int kMostThreads = 256;  // of a CTA

struct AppendParams {
  Kv8Layer c;
  Kv8Entries e;
  const __half *k, *v;
  const int* positions;
  const int* refs;       // how many table entries name a page, or nullptr
  long long batch_stride, token_stride, head_stride;
  int unit, unit_shift;  // threads of a unit: a power of two, 32 .. 256
  int heads_shift;       // units of a CTA: neighbouring heads
  float minus_zero;
  DeviceStatus* status;
};

// Whether n tokens from position pos0 on have a place in a row of the page table.
__device__ __forceinline__ bool fits(const Kv8Layer& c, int pos0, int n) {
  return pos0 >= 0 && (long long)pos0 + n <= ((long long)c.max_pages << c.page_shift);
}

// Codes of a block whose scale grows.  The ratio is at most 1 (to rounding); a code -128 that somebody else wrote becomes -127.
template <int TYPE>
__device__ __forceinline__ uint32_t encode_held(const float (&f)[4], float ratio) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = TYPE == LIGER_KV8_INT8 ? fmaxf(f[i] * ratio, -127.0f) : f[i] * ratio;
  return kv8_encode4<TYPE>(y[0], y[1], y[2], y[3]);
}

// Eight values times the reciprocal, in pairs, and rounded (how: kv8_encode4).  The product is an fma with -0 that the compiler cannot
// see: it would join a product and the rounding addition into one fma, which rounds once where the definition rounds twice.
template <int TYPE>
__device__ __forceinline__ uint2 encode_new(const uint4& x, float back, float minus_zero) {
  const uint32_t h[4] = {x.x, x.y, x.z, x.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    float2 y;
    asm("{\n\t.reg .b64 v, b, z;\n\tmov.b64 v, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\tfma.rn.f32x2 v, v, b, z;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "=f"(y.x), "=f"(y.y)
        : "f"(f.x), "f"(f.y), "f"(back), "f"(minus_zero));
    if (TYPE == LIGER_KV8_INT8) {
      asm("{\n\t.reg .b64 v, b;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tadd.rn.f32x2 v, v, b;\n\tmov.b64 {%0, %1}, v;\n\t}"
          : "+f"(y.x), "+f"(y.y)
          : "f"(kWholeNumbers));
      c[i] = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040);
    } else {
      uint16_t pair;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(y.y), "f"(y.x));
      c[i] = pair;
    }
  }
  return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}

// Grid: (2 * groups of heads, blocks that an entry can touch, entries); a CTA has as many units of neighbouring heads, whose source
// rows are neighbours, as fit.  Bound by HBM as to what it moves, and nearly as much by instructions: no division for a unit's place
// (45 -> 36 us for 2256 tokens x 96 heads of 128, int8), two products or roundings in one instruction, the values' loads before the
// table's answer is looked at, small CTAs (-> 33.8).  That is 5.1 TB/s, 78 % of the copy rate; a CTA has one phase of loads and one of stores.
template <int D, int TYPE, int U>
__global__ void __launch_bounds__(kMostThreads) kv8_append_kernel(const AppendParams p) {
  constexpr int kPieces = D / 8;  // 16-byte pieces of a source row
  __shared__ uint32_t s_max[kMostThreads / 32];
  wait_for_stream();
  const int b = blockIdx.z;
  int n, row0;
  const bool rows_ok = kv8_rows(p.e, b, n, row0);
  const int slot = kv8_slot(p.e, b);
  const int pos0 = kv8_ld(p.positions + b);
  const bool lead = blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0;
  if (!rows_ok || n == 0) {
    if (lead && !rows_ok) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAppend, b, 0);
    return;
  }
  if (slot < 0 || slot >= p.c.slots || !fits(p.c, pos0, n)) {
    if (lead) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAppend + 1, b, (unsigned)slot);
    return;
  }
  if (p.e.slots) {  // an earlier entry of the same slot that brings tokens, and is not itself left out, has it
    bool dup = false;
    for (int j = threadIdx.x; j < b; j += blockDim.x)
      if (kv8_ld(p.e.slots + j) == slot) {
        int n_j, row0_j;
        dup |= kv8_rows(p.e, j, n_j, row0_j) && n_j > 0 && fits(p.c, kv8_ld(p.positions + j), n_j);
      }
    if (__syncthreads_or(dup)) {
      if (lead) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAppend + 2, b, (unsigned)slot);
      return;
    }
  }
  const int t = threadIdx.x & (p.unit - 1);
  const int is_v = blockIdx.x & 1, blk = blockIdx.y;
  const int head = ((blockIdx.x >> 1) << p.heads_shift) + (threadIdx.x >> p.unit_shift);
  const int block0 = pos0 >> p.c.block_shift;            // the first block that is touched
  const int start = (block0 + blk) << p.c.block_shift;   // this unit's first position
  if (start >= pos0 + n) return;  // the whole CTA
  const bool wanted = head < p.c.kv_heads;
  const int page = wanted ? kv8_ld(p.c.table + (size_t)slot * p.c.max_pages + (start >> p.c.page_shift)) : -1;
  const __half* src = (is_v ? p.v : p.k) + (p.e.q_offsets ? (long long)row0 * p.token_stride : (long long)b * p.batch_stride) +
                      (long long)head * p.head_stride;
  const int held = pos0 - start;      // tokens that the block held before, where positive
  const int end = pos0 + n - start;   // rows [max(held, 0), end) are new

  // the thread's pieces: piece `piece` of rows r0, r0 + rows_u, ...
  const int piece = t % kPieces, r0 = t / kPieces, rows_u = p.unit / kPieces;
  const int r_end = min(end, 1 << p.c.block_shift);
  const bool full = wanted && held <= 0 && end >= (1 << p.c.block_shift);  // the usual block: no row has to be asked
  uint4 x[U];
  __half2 hm = __half2half2(__ushort_as_half(0));
  {
    const __half* at = src + (long long)(start + r0 - pos0) * p.token_stride + piece * 8;
    const long long step = (long long)rows_u * p.token_stride;
    if (full) {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = __ldcs(reinterpret_cast<const uint4*>(at + u * step));
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * rows_u;
        x[u] = make_uint4(0, 0, 0, 0);
        if (wanted && r >= held && r < r_end) x[u] = __ldcs(reinterpret_cast<const uint4*>(at + u * step));
      }
    }
  }
  bool active = wanted;
  if (active && (page < 0 || page >= p.c.num_pages)) {  // asked only now, so that the values are under way before the table has answered
    if (t == 0) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAppend + 3, b, (unsigned)page);
    active = false;
  } else if (active && p.refs && kv8_ld(p.refs + page) > 1) {  // another slot reads it, too (to ask costs 0.2 us of a token each, 2 us of the prompts above)
    if (t == 0) report_failure(p.status, LIGER_DEV_BAD_INDEX, kKv8AtAppend + 4, b, (unsigned)page);
    active = false;
  }
  const int inside = start & ((1 << p.c.page_shift) - 1);
  const size_t page_head = active ? (size_t)page * p.c.kv_heads + head : 0;
  uint8_t* codes = (is_v ? p.c.v : p.c.k) + ((page_head << p.c.page_shift) + inside) * D;
  float* scale = (is_v ? p.c.vs : p.c.ks) + (page_head << (p.c.page_shift - p.c.block_shift)) + (inside >> p.c.block_shift);
  const bool goes_on = active && held > 0;
  const float s_old = goes_on ? *scale : 0.0f;

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const __half2* h = reinterpret_cast<const __half2*>(&x[u]);
#pragma unroll
    for (int j = 0; j < 4; ++j) hm = __hmax2_nan(hm, __habs2(h[j]));
  }
  const uint32_t hb = *reinterpret_cast<const uint32_t*>(&hm);
  uint32_t mx = __reduce_max_sync(0xffffffffu, max(hb & 0xffffu, hb >> 16));
  if (p.unit > 32) {  // the same for the whole grid
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) s_max[warp] = mx;
    __syncthreads();
    const int w0 = warp & ~(p.unit / 32 - 1);
    for (int i = 0; i < p.unit / 32; ++i) mx = max(mx, s_max[w0 + i]);
  }
  if (!active) return;
  const float amax = __half2float(__ushort_as_half((unsigned short)mx));
  const float now = amax * (1.0f / (TYPE == LIGER_KV8_INT8 ? 127.0f : 448.0f));
  const float s = goes_on && !(now > s_old) && now == now ? s_old : now;  // a scale that is NaN stays
  const bool finite = s > 0.0f && s <= 3.0e38f;
  const float back = finite ? 1.0f / s : 0.0f;
  if (goes_on && !(s == s_old)) {
    const float ratio = s_old * back;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * rows_u;
      if (r < held && r < (1 << p.c.block_shift)) {
        uint2* at = reinterpret_cast<uint2*>(codes + (size_t)r * D + piece * 8);
        uint2 c = make_uint2(0, 0);
        if (finite) {
          c = *at;
          float f[4];
          kv8_decode4<TYPE>(c.x, f);
          c.x = encode_held<TYPE>(f, ratio);
          kv8_decode4<TYPE>(c.y, f);
          c.y = encode_held<TYPE>(f, ratio);
        }
        *at = c;
      }
    }
  }
  uint8_t* out = codes + r0 * D + piece * 8;
  if (full && finite) {
#pragma unroll
    for (int u = 0; u < U; ++u) *reinterpret_cast<uint2*>(out + u * rows_u * D) = encode_new<TYPE>(x[u], back, p.minus_zero);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * rows_u;
      if (r >= held && r < r_end) *reinterpret_cast<uint2*>(out + u * rows_u * D) = finite ? encode_new<TYPE>(x[u], back, p.minus_zero) : make_uint2(0, 0);
    }
  }
  if (t == 0) *scale = s;
}

template <int D, int U>
int launch_append(const AppendParams& p, int blocks, int type, cudaStream_t stream) {
  const int heads_cta = 1 << p.heads_shift;
  const dim3 grid(2 * ((p.c.kv_heads + heads_cta - 1) / heads_cta), blocks, p.e.batch);
  return launch_early("kv8_append_kernel", type == LIGER_KV8_INT8 ? kv8_append_kernel<D, LIGER_KV8_INT8, U> : kv8_append_kernel<D, LIGER_KV8_E4M3, U>,
                      grid, p.unit << p.heads_shift, 0, stream, p);
}

}  // namespace
}  // namespace liger

using namespace liger;

extern "C" int liger_kv8_append(const liger_kv8_cache* cache, const liger_kv8_append_args* a, void* stream) {
  if (!a) return set_error(LIGER_ERR_INVALID, "kv8_append: args is NULL");
  int rc = kv8_check("kv8_append", cache, a->layer);
  if (rc != LIGER_OK) return rc;
  if (a->layer < 0) return set_error(LIGER_ERR_INVALID, "kv8_append: layer %d", a->layer);
  if (!a->k || !a->v || !a->positions) return set_error(LIGER_ERR_INVALID, "kv8_append: a pointer is NULL");
  if (((uintptr_t)a->k | (uintptr_t)a->v) & 15u) return set_error(LIGER_ERR_INVALID, "kv8_append: k / v must be 16-byte aligned");
  if (((uintptr_t)a->positions | (uintptr_t)a->slots) & 3u)
    return set_error(LIGER_ERR_INVALID, "kv8_append: positions and slots must be 4-byte aligned");
  rc = kv8_check_tokens("kv8_append", a->q_offsets, a->batch, a->q_len, a->total_tokens, a->batch_stride, a->token_stride, a->head_stride);
  if (rc != LIGER_OK) return rc;
  const DeviceInfo* dev = current_device();
  if (!dev) return LIGER_ERR_CUDA;
  AppendParams p{};
  p.c = kv8_layer(cache, a->layer);
  p.e = Kv8Entries{a->q_offsets, a->slots, a->batch, a->q_len, a->total_tokens};
  p.k = (const __half*)a->k;
  p.v = (const __half*)a->v;
  p.positions = a->positions;
  p.refs = cache->page_refs;
  p.batch_stride = a->batch_stride;
  p.token_stride = a->token_stride;
  p.head_stride = a->head_stride;
  p.minus_zero = -0.0f;
  p.status = dev->status_dev;
  // q_len tokens that begin at the last place of a block touch this many
  const long long blocks = ((long long)a->q_len + cache->scale_block - 2) / cache->scale_block + 1;
  if (blocks > 65535) return set_error(LIGER_ERR_UNSUPPORTED, "kv8_append: q_len %d touches more than 65535 blocks of %d tokens", a->q_len, cache->scale_block);
  const int pieces = cache->scale_block * (cache->head_dim / 8);
  p.unit = pieces / 8 < 32 ? 32 : pieces / 8;
  p.unit_shift = 31 - __builtin_clz(p.unit);
  p.heads_shift = p.unit < 128 ? 7 - p.unit_shift : 0;  // 128 threads: 33.8 us; 256 take 0.9 more, 64 take 1.5 more
  cudaStream_t s = (cudaStream_t)stream;
  if (cache->head_dim == 128) return launch_append<128, 8>(p, (int)blocks, cache->type, s);
  return pieces / 8 < 32 ? launch_append<64, 4>(p, (int)blocks, cache->type, s) : launch_append<64, 8>(p, (int)blocks, cache->type, s);
}
