// The paged 8-bit key/value cache as its kernels see it: one layer's arrays, the entries (sequences) of a call, and the
// conversions between fp16 / fp32 and the two code types.
#pragma once
#include <atomic>

#include "runtime.h"

namespace liger {

// One layer of a liger_kv8_cache.  Page p, head h, token t of the page: codes at (((p * kv_heads + h) << page_shift) + t) *
// head_dim, its scale at ((p * kv_heads + h) << (page_shift - block_shift)) + (t >> block_shift).
struct Kv8Layer {
  uint8_t *k, *v;
  float *ks, *vs;
  const int* table;
  int num_pages, kv_heads, page_shift, block_shift, slots, max_pages;
};

// The entries of a call, as append and attention share them.
struct Kv8Entries {
  const int* q_offsets;  // [batch + 1] or nullptr
  const int* slots;      // [batch] or nullptr
  int batch, q_len, total_tokens;
};

// Locations in the sticky device status
constexpr unsigned kKv8AtAppend = 0x500u, kKv8AtAttention = 0x510u, kKv8AtPages = 0x520u;

// Checks the parts of a cache that every operator uses; `layer` < 0: the call is about all layers.
int kv8_check(const char* what, const liger_kv8_cache* c, int layer);
Kv8Layer kv8_layer(const liger_kv8_cache* c, int layer);
// Checks batch, q_len, offsets and strides of the new tokens of a call.
int kv8_check_tokens(const char* what, const int* q_offsets, int batch, int q_len, int total_tokens, long long batch_stride,
                     long long token_stride, long long head_stride);

#ifdef __CUDACC__

// Every kernel of the cache is launched while its predecessor on the stream may still run (launch_early), waits for it here
// before it touches memory, and lets its successor be launched.  All CTAs wait, also those that have nothing to do: a successor
// counts on a kernel's end for the end of all that came before it.
__device__ __forceinline__ void wait_for_stream() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// What may have been written by the predecessor is read with ordinary loads: the read-only path is for data that does not change
// while the grid lives, and the grid begins before its predecessor ends.
template <typename T>
__device__ __forceinline__ T kv8_ld(const T* p) { return *p; }

template <typename... Params, typename... Args>
int launch_early(const char* what, void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(LIGER_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
  }
  return LIGER_OK;
}
// Allows `kernel` this much shared memory, once on each device (the call costs about 2 us); `done` is the kernel's own.
template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes, const DeviceInfo* dev, std::atomic<unsigned long long>& done) {
  const unsigned long long bit = 1ull << (dev->device & 63);
  if (done.load(std::memory_order_relaxed) & bit) return LIGER_OK;
  LIGER_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return LIGER_OK;
}

// New tokens of entry b: their number, and the first one's row among all tokens of the call.  False: the offsets are not a
// run of at most q_len rows inside [0, total_tokens).
__device__ __forceinline__ bool kv8_rows(const Kv8Entries& e, int b, int& n, int& row0) {
  if (e.q_offsets == nullptr) {
    n = e.q_len;
    row0 = b * e.q_len;
    return true;
  }
  const int lo = kv8_ld(e.q_offsets + b), hi = kv8_ld(e.q_offsets + b + 1);
  if (lo < 0 || hi < lo || hi > e.total_tokens || hi - lo > e.q_len) {
    n = 0;
    row0 = 0;
    return false;
  }
  n = hi - lo;
  row0 = lo;
  return true;
}

__device__ __forceinline__ int kv8_slot(const Kv8Entries& e, int b) { return e.slots ? kv8_ld(e.slots + b) : b; }

// ---- codes ----------------------------------------------------------------------------------------------------------------
// 1.5 * 2^23 + x: the sum's last place is 1, so the addition rounds x to a whole number (to even at ties) and leaves it in the
// low bits.  A conversion instruction would do it at an eighth of the rate.  |x| is below 128 (kv8_append_kernel).
constexpr float kWholeNumbers = 12582912.0f;
// fp32 -> code, round to nearest even; e4m3 saturates, int8 wants what rounds to -127 .. 127
template <int TYPE>
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d) {
  if (TYPE == LIGER_KV8_INT8) {
    const float whole = kWholeNumbers;
    const uint32_t ia = __float_as_uint(__fadd_rn(a, whole)), ib = __float_as_uint(__fadd_rn(b, whole));
    const uint32_t ic = __float_as_uint(__fadd_rn(c, whole)), id = __float_as_uint(__fadd_rn(d, whole));
    return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
  } else {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  }
}

// Two codes -> half2, exact for both types (127 needs 7 bits, an e4m3 number 4 bits between 2^-9 and 448).  `w` holds the pair
// in its lower (HIGH = 0) or upper 16 bits; int8 codes must have been biased by kv8_bias().
template <int TYPE>
__device__ __forceinline__ uint32_t kv8_bias(uint32_t w) {
  return TYPE == LIGER_KV8_INT8 ? w ^ 0x80808080u : w;
}
template <int TYPE, int HIGH>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w) {
  uint32_t r;
  if (TYPE == LIGER_KV8_INT8) {
    // code + 128 in the low byte of the half 1024 + (code + 128); minus 1152 is exact
    r = __byte_perm(w, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
    r = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const uint16_t p = HIGH ? (uint16_t)(w >> 16) : (uint16_t)w;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(p));
  }
  return r;
}
template <int TYPE>
__device__ __forceinline__ void kv8_decode4(uint32_t w, float (&f)[4]) {
  const uint32_t b = kv8_bias<TYPE>(w);
  const uint32_t lo = kv8_pair<TYPE, 0>(b), hi = kv8_pair<TYPE, 1>(b);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
}

#endif

}  // namespace liger
