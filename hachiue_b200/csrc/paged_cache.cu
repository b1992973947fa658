// paged_cache.cu - rows into and out of the paged 4-bit cache: the rotated
// append (hcu_rope_append_paged) and the gather (hcu_read_paged).
//
// Both move each row once and are bound by HBM for prompts and by launch
// latency for single tokens.  One warp takes one row of one head; lane l holds
// elements 4l .. 4l + 3 of each 128, so a Q4_0 block is eight lanes, a value
// halfword is one lane's codes and a key word those of two.
#include "paged.cuh"

namespace hcu {
namespace {

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* cos_tab;
  const float* sin_tab;
  const int32_t* positions;
  const int64_t* slots;
  void* q_out;
  void* k_out;
  PagedKV kv;
  long long q_stride, k_stride, v_stride, n_slots;
  int n, H, half, table_rows;
  uint32_t* status;
};

// floor(x / d + 8.5) held within 0..15, exactly, without a division: the f32
// estimate is off by at most one level next to a border, and the borders
// (c - 8.5) * d and (c - 7.5) * d of a level are products of an 11-bit and a
// 5-bit number, exact in f32, so two compares put it right.  y is x times the
// sign of d, a is |d| (an f16 value above 0), inv about 1 / a.
__device__ __forceinline__ uint32_t q4_code(float y, float a, float inv) {
  float c = floorf(fminf(fmaxf(fmaf(y, inv, 8.5f), 0.f), 15.f));
  if ((c - 8.5f) * a > y) c -= 1.f;
  if ((c - 7.5f) * a <= y) c += 1.f;
  return (uint32_t)(int)fminf(fmaxf(c, 0.f), 15.f);
}

// Quantises the four elements of each lane: a block is the eight lanes of
// equal lane / 8.  Returns the lane's four codes (element 0 lowest) and the
// block's scale.
__device__ __forceinline__ uint32_t q4_block(const float (&x)[4], int lane, __half* scale) {
  uint32_t top = 0;
  float m = x[0];  // the lane's first element of the lane's largest magnitude
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const uint32_t b = __float_as_uint(x[c]) & 0x7fffffffu;
    if (b > top) {
      top = b;
      m = x[c];
    }
  }
  uint32_t all = top;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) all = max(all, __shfl_xor_sync(0xffffffffu, all, o));
  const uint32_t same = __ballot_sync(0xffffffffu, top == all);
  const int first = (lane & 24) + __ffs((same >> (lane & 24)) & 0xffu) - 1;
  m = __shfl_sync(0xffffffffu, m, first);
  const __half d = __float2half_rn(fminf(fmaxf(m * -0.125f, -65504.f), 65504.f));
  *scale = d;
  const float df = __half2float(d), a = fabsf(df);
  if (a == 0.f) return 0x8888u;
  const float inv = __fdiv_rn(1.f, a);
  const uint32_t sign = __float_as_uint(df) & 0x80000000u;
  uint32_t code = 0;
#pragma unroll
  for (int c = 0; c < 4; c++) code |= q4_code(__uint_as_float(__float_as_uint(x[c]) ^ sign), a, inv) << (4 * c);
  return code;
}

template <typename T, int DH>
__global__ void __launch_bounds__(256) rope_append_kernel(const AppendArgs a) {
  constexpr int NJ = DH / 128, NB = DH / 32;
  const int lane = threadIdx.x & 31, heads = a.H + 2 * a.kv.KV;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (long long)a.n * heads) return;
  const int i = (int)(row / heads), r = (int)(row % heads);
  const long long slot = a.slots[i];
  if (slot < 0) return;
  const int pos = a.half ? a.positions[i] : 0;
  if (slot >= a.n_slots || (a.half && (pos < 0 || pos >= a.table_rows))) {
    if (r == 0 && lane == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
    return;
  }
  const int kind = r < a.H ? 0 : (r < a.H + a.kv.KV ? 1 : 2);  // q, k, v
  const int g = kind == 0 ? r : (kind == 1 ? r - a.H : r - a.H - a.kv.KV);
  const T* src = kind == 0   ? static_cast<const T*>(a.q) + i * a.q_stride
                 : kind == 1 ? static_cast<const T*>(a.k) + i * a.k_stride
                             : static_cast<const T*>(a.v) + i * a.v_stride;
  src += (long long)g * DH;
  float x[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; j++) load4(src + 128 * j + 4 * lane, x[j]);
  if (kind < 2) {
    // The partner elements come from memory again (the row is in L1), so any
    // rotaryDim that is a multiple of 8 takes the same path.
    const float* ct = a.cos_tab + (long long)pos * a.half;
    const float* st = a.sin_tab + (long long)pos * a.half;
    float w[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int e = 128 * j + 4 * lane;
      if (e < 2 * a.half) load4(src + (e < a.half ? e + a.half : e - a.half), w[j]);
    }
    __syncwarp();  // in place: the row has been read before any lane writes
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int e = 128 * j + 4 * lane;
      if (e < 2 * a.half) {
        const bool low = e < a.half;
        float c[4], s[4];
        load4(ct + (low ? e : e - a.half), c);
        load4(st + (low ? e : e - a.half), s);
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const float sg = low ? -s[t] : s[t];
          if (kind == 0)
            x[j][t] = fmaf(x[j][t], c[t], w[j][t] * sg);
          else  // the products of two f32 values are exact in f64
            x[j][t] = (float)__dadd_rn(__dmul_rn(x[j][t], c[t]), __dmul_rn(w[j][t], sg));
        }
      }
    }
    T* dst = kind == 0 ? static_cast<T*>(a.q_out) : static_cast<T*>(a.k_out);
    if (dst) {
      dst += ((long long)i * (kind == 0 ? a.H : a.kv.KV) + g) * DH;
#pragma unroll
      for (int j = 0; j < NJ; j++) store4(dst + 128 * j + 4 * lane, x[j]);
    }
    if (kind == 0) return;
  }
  const long long at = paged_row(a.kv, slot >> a.kv.page_log2, g, (int)(slot & ((1 << a.kv.page_log2) - 1)));
  uint8_t* codes = (kind == 1 ? a.kv.k : a.kv.v) + at * (DH / 2);
  __half* scales = (kind == 1 ? a.kv.ks : a.kv.vs) + at * NB;
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int b = 4 * j + (lane >> 3), l = lane & 7;  // block, lane in the block
    __half d;
    const uint32_t c = q4_block(x[j], lane, &d);
    if (kind == 1) {
      const uint32_t hi = __shfl_xor_sync(0xffffffffu, c, 1);
      if (!(l & 1)) *reinterpret_cast<uint32_t*>(codes + ((l >> 1) * NB + b) * 4) = c | hi << 16;
    } else {
      *reinterpret_cast<uint16_t*>(codes + (l * NB + b) * 2) = (uint16_t)c;
    }
    if (l == 0) scales[b] = d;
  }
}

struct ReadArgs {
  const int64_t* slots;
  PagedKV kv;
  long long n_slots;
  int n;
  void* k_out;
  void* v_out;
  uint32_t* status;
};

template <typename T, int DH>
__global__ void __launch_bounds__(256) read_paged_kernel(const ReadArgs a) {
  constexpr int NJ = DH / 128, NB = DH / 32;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (long long)a.n * a.kv.KV * 2) return;
  const int i = (int)(row / (2 * a.kv.KV)), r = (int)(row % (2 * a.kv.KV));
  const long long slot = a.slots[i];
  if (slot < 0) return;
  if (slot >= a.n_slots) {
    if (r == 0 && lane == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
    return;
  }
  const bool key = r < a.kv.KV;
  const int g = key ? r : r - a.kv.KV;
  const long long at = paged_row(a.kv, slot >> a.kv.page_log2, g, (int)(slot & ((1 << a.kv.page_log2) - 1)));
  const uint8_t* codes = (key ? a.kv.k : a.kv.v) + at * (DH / 2);
  const __half* scales = (key ? a.kv.ks : a.kv.vs) + at * NB;
  T* dst = static_cast<T*>(key ? a.k_out : a.v_out) + ((long long)i * a.kv.KV + g) * DH;
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int b = 4 * j + (lane >> 3), l = lane & 7;
    const uint32_t c = key ? *reinterpret_cast<const uint16_t*>(codes + ((l >> 1) * NB + b) * 4 + (l & 1) * 2)
                           : *reinterpret_cast<const uint16_t*>(codes + (l * NB + b) * 2);
    const float d = __half2float(scales[b]);
    float x[4];
#pragma unroll
    for (int t = 0; t < 4; t++) x[t] = (float)((int)((c >> (4 * t)) & 15u) - 8) * d;
    store4(dst + 128 * j + 4 * lane, x);
  }
}

// Calls f with a null pointer of the element type of `dtype`.
template <typename F>
int with_dtype(const char* op, uint32_t dtype, F&& f) {
  switch (dtype) {
    case HCU_DT_F32: return f(static_cast<float*>(nullptr));
    case HCU_DT_F16: return f(static_cast<__half*>(nullptr));
    case HCU_DT_BF16: return f(static_cast<__nv_bfloat16*>(nullptr));
  }
  return fail(HCU_EINVAL, "%s: unknown dtype %u", op, dtype);
}

template <typename T>
int launch_append(hcu_context* h, const AppendArgs& a, int dh) {
  const long long blocks = ((long long)a.n * (a.H + 2 * a.kv.KV) + 7) / 8;
  if (blocks > 0x7fffffffLL) return fail(HCU_EINVAL, "hcu_rope_append_paged: too many rows");
  if (dh == 128) rope_append_kernel<T, 128><<<(unsigned)blocks, 256, 0, h->stream>>>(a);
  else rope_append_kernel<T, 256><<<(unsigned)blocks, 256, 0, h->stream>>>(a);
  return after_launch("hcu_rope_append_paged: launch");
}

template <typename T>
int launch_read(hcu_context* h, const ReadArgs& a, int dh) {
  const long long blocks = ((long long)a.n * a.kv.KV * 2 + 7) / 8;
  if (blocks > 0x7fffffffLL) return fail(HCU_EINVAL, "hcu_read_paged: too many rows");
  if (dh == 128) read_paged_kernel<T, 128><<<(unsigned)blocks, 256, 0, h->stream>>>(a);
  else read_paged_kernel<T, 256><<<(unsigned)blocks, 256, 0, h->stream>>>(a);
  return after_launch("hcu_read_paged: launch");
}

}  // namespace
}  // namespace hcu

using hcu::fail;

extern "C" int hcu_rope_append_paged(hcu_handle h, const hcu_rope_append_params* p, const void* q, const void* k,
                                     const void* v, const float* cos_tab, const float* sin_tab,
                                     const int32_t* positions, const int64_t* slots, void* q_out, void* k_out,
                                     const hcu_paged_kv* kv) {
  const char* op = "hcu_rope_append_paged";
  hcu::DeviceScope scope;
  HCU_TRY(hcu::begin_op(h, op));
  hcu::AppendArgs a{};
  if (!p) return fail(HCU_EINVAL, "%s: null params", op);
  HCU_TRY(hcu::check_paged(op, kv, &a.kv));
  const int eb = hcu::dtype_bytes(p->dtype);
  if (!eb) return fail(HCU_EINVAL, "%s: unknown dtype %u", op, p->dtype);
  if (p->n > 0x7fffffffu || p->H > 65535u) return fail(HCU_EINVAL, "%s: n or H too large", op);
  if (p->rotaryDim % 8 || p->rotaryDim > kv->Dh)
    return fail(HCU_EINVAL, "%s: rotaryDim (%u) must be a multiple of 8, at most Dh (%u)", op, p->rotaryDim, kv->Dh);
  if (p->n == 0) return HCU_OK;
  if (!k || !v || !slots) return fail(HCU_EINVAL, "%s: null k, v or slots", op);
  if (p->H && (!q || !q_out)) return fail(HCU_EINVAL, "%s: H queries need q and q_out", op);
  if (p->rotaryDim && (!cos_tab || !sin_tab || !positions))
    return fail(HCU_EINVAL, "%s: a rotation needs cos, sin and positions", op);
  if (p->table_rows > 0x7fffffffu) return fail(HCU_EINVAL, "%s: table_rows too large", op);
  const uint64_t qs = p->q_row_stride ? p->q_row_stride : (uint64_t)p->H * kv->Dh;
  const uint64_t ks = p->k_row_stride ? p->k_row_stride : (uint64_t)kv->KV * kv->Dh;
  const uint64_t vs = p->v_row_stride ? p->v_row_stride : (uint64_t)kv->KV * kv->Dh;
  if (qs % 4 || ks % 4 || vs % 4) return fail(HCU_EINVAL, "%s: row strides must be multiples of 4 elements", op);
  if (qs < (uint64_t)p->H * kv->Dh || ks < (uint64_t)kv->KV * kv->Dh || vs < (uint64_t)kv->KV * kv->Dh)
    return fail(HCU_EINVAL, "%s: a row stride is shorter than its row", op);
  if ((qs | ks | vs) >> 40) return fail(HCU_EINVAL, "%s: a row stride is too large", op);
  const uintptr_t rows = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         reinterpret_cast<uintptr_t>(k_out) |
                         (p->H ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0);
  if (rows % (4 * eb)) return fail(HCU_EINVAL, "%s: rows must be aligned to four elements", op);
  if (p->rotaryDim && ((reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab)) % 16))
    return fail(HCU_EINVAL, "%s: cos and sin must be 16-byte aligned", op);
  if (p->H && q_out == q && qs != (uint64_t)p->H * kv->Dh)
    return fail(HCU_EINVAL, "%s: q_out may be q itself only where q is dense", op);
  if (k_out == k && ks != (uint64_t)kv->KV * kv->Dh)
    return fail(HCU_EINVAL, "%s: k_out may be k itself only where k is dense", op);
  a.q = q;
  a.k = k;
  a.v = v;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.positions = positions;
  a.slots = slots;
  a.q_out = q_out;
  a.k_out = k_out;
  a.q_stride = (long long)qs;
  a.k_stride = (long long)ks;
  a.v_stride = (long long)vs;
  a.n_slots = (long long)kv->n_pages << a.kv.page_log2;
  a.n = (int)p->n;
  a.H = (int)p->H;
  a.half = (int)p->rotaryDim / 2;
  a.table_rows = (int)p->table_rows;
  a.status = h->dev_status;
  return hcu::with_dtype(op, p->dtype, [&](auto* t) {
    return hcu::launch_append<std::remove_pointer_t<decltype(t)>>(h, a, (int)kv->Dh);
  });
}

extern "C" int hcu_read_paged(hcu_handle h, uint32_t n, uint32_t dtype, const int64_t* slots, const hcu_paged_kv* kv,
                              void* k_out, void* v_out) {
  const char* op = "hcu_read_paged";
  hcu::DeviceScope scope;
  HCU_TRY(hcu::begin_op(h, op));
  hcu::ReadArgs a{};
  HCU_TRY(hcu::check_paged(op, kv, &a.kv));
  const int eb = hcu::dtype_bytes(dtype);
  if (!eb) return fail(HCU_EINVAL, "%s: unknown dtype %u", op, dtype);
  if (n > 0x7fffffffu) return fail(HCU_EINVAL, "%s: n too large", op);
  if (n == 0) return HCU_OK;
  if (!slots || !k_out || !v_out) return fail(HCU_EINVAL, "%s: null slots or output", op);
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % (4 * eb))
    return fail(HCU_EINVAL, "%s: outputs must be aligned to four elements", op);
  a.slots = slots;
  a.n_slots = (long long)kv->n_pages << a.kv.page_log2;
  a.n = (int)n;
  a.k_out = k_out;
  a.v_out = v_out;
  a.status = h->dev_status;
  return hcu::with_dtype(op, dtype, [&](auto* t) {
    return hcu::launch_read<std::remove_pointer_t<decltype(t)>>(h, a, (int)kv->Dh);
  });
}
