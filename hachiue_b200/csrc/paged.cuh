// paged.cuh - the paged 4-bit KV cache (hcu_paged_kv, HCU_KV_Q4_0) as its
// append, read and attention kernels see it, and the activation types.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "context.h"

namespace hcu {

// Four consecutive elements of an activation row, as f32 (16 or 8 bytes of memory).
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void load4(const __half* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = f16x2_to_f2(v.x), b = f16x2_to_f2(v.y);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = bf16_lo(v.x), x[1] = bf16_hi(v.x), x[2] = bf16_lo(v.y), x[3] = bf16_hi(v.y);
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__half* p, const float (&x)[4]) {
  const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Eight elements: two 16-byte accesses of f32, one of the 16-bit types.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (std::is_same<T, __half>::value) {
      const float2 f = f16x2_to_f2(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Packed f32 pairs: one instruction for two lanes of a 64-bit register pair.
__device__ __forceinline__ uint64_t f2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void f2_get(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// 16 bytes from global into shared memory by the asynchronous copy unit; nothing is read and zeros are written unless `there`.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The device view of an hcu_paged_kv.
struct PagedKV {
  uint8_t* k;
  uint8_t* v;
  __half* ks;
  __half* vs;
  int page_log2, n_pages, KV;
};

// Row index of `offset` in page `page` for KV head g (rows of Dh / 2 code bytes, Dh / 32 scales).
__device__ __forceinline__ long long paged_row(const PagedKV& c, long long page, int g, int offset) {
  return ((page * c.KV + g) << c.page_log2) + offset;
}

// Checks the cache's geometry and fills the device view (host).
inline int check_paged(const char* op, const hcu_paged_kv* kv, PagedKV* out) {
  if (!kv) return fail(HCU_EINVAL, "%s: null cache", op);
  if (kv->format != HCU_KV_Q4_0) return fail(HCU_EUNSUPPORTED, "%s: paged cache format %u (built: HCU_KV_Q4_0)", op, kv->format);
  if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
    return fail(HCU_EINVAL, "%s: page_size (%u) must be 16, 32, 64, 128 or 256", op, kv->page_size);
  if (kv->n_pages == 0 || kv->KV == 0) return fail(HCU_EINVAL, "%s: n_pages and KV must be positive", op);
  if (kv->n_pages > 0x7fffffffu || kv->KV > 65535u) return fail(HCU_EINVAL, "%s: n_pages or KV too large", op);
  if (kv->Dh != 128 && kv->Dh != 256) return fail(HCU_EUNSUPPORTED, "%s: Dh=%u (built: 128, 256)", op, kv->Dh);
  if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale) return fail(HCU_EINVAL, "%s: null cache buffer", op);
  if ((reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v) |
       reinterpret_cast<uintptr_t>(kv->k_scale) | reinterpret_cast<uintptr_t>(kv->v_scale)) % 16)
    return fail(HCU_EINVAL, "%s: cache buffers must be 16-byte aligned", op);
  int lg = 4;
  while ((1u << lg) < kv->page_size) lg++;
  *out = PagedKV{static_cast<uint8_t*>(kv->k),       static_cast<uint8_t*>(kv->v),
                 static_cast<__half*>(kv->k_scale),  static_cast<__half*>(kv->v_scale),
                 lg,                                 (int)kv->n_pages,
                 (int)kv->KV};
  return HCU_OK;
}

inline int dtype_bytes(uint32_t dt) { return dt == HCU_DT_F32 ? 4 : (dt == HCU_DT_F16 || dt == HCU_DT_BF16) ? 2 : 0; }

}  // namespace hcu
