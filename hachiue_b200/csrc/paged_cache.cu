// paged_cache.cu - rows into and out of the paged 4-bit cache: the rotated
// append (hcu_rope_append_paged) and the gather (hcu_read_paged).
//
// Both move each row once, so HBM is their floor for prompts (launch latency for
// single tokens); the arithmetic per 4-bit code is what stands above it.
//  * Append: a block per token, so that its cos and sin values are loaded once
//    into registers for all of its rows; eight elements per lane, a row of 128
//    being half a warp.  A Q4_0 block is then four lanes, a lane's codes one word of
//    a key row or two halfwords of a value row.  For prompts four blocks per SM walk
//    the tokens, each with the next one's rows on their way into L2 (a block per
//    token spent its life waiting for its slot, then its angles, then its rows: 76
//    against 65 us below).  8192 tokens of 32 query, 8 key and 8 value heads of 128,
//    bf16: 65 us (L2 flushed), 181 MB at 2.8 TB/s, of which the values' and keys' codes
//    take 40: 370 instructions per warp and two rows, at 70 % of the issue rate.
//  * Read: eight bytes of codes per lane, so that a warp has four rows of 128 of
//    both tensors in flight, and writes whole 32-byte sectors.  16384 rows of 8 heads
//    of 128 to bf16: 18 us, 86 MB at 4.7 TB/s, ALU pipe 70 %.
#include <algorithm>

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

// floor(x / d + 8.5) held within 0..15, exactly, without a division.  d is an
// f16 value other than 0 and inv about 1 / d; y is x times the sign of d, a is |d|.
//
// q4_codes: x * inv + 8 + 2^-18, rounded to the nearest integer.  The sum is
// off by less than 2^-19 (inv by an ulp, the sum by half of one), so a border
// goes to the level above it, as it should, and only a y less than 2^-17 a
// below a border can be taken for it.  There is none among 16-bit inputs: y is a
// multiple of 2^-12 a there, and so is a border (an 11-bit number times an odd
// multiple of a half).  Where y is any f32 number such a one is looked for, and
// q4_code puts it right by comparing with the borders (c - 8.5) a and (c - 7.5) a,
// products of an 11-bit and a 5-bit number, exact in f32.
__device__ __forceinline__ uint32_t q4_code(float y, float a, float inv) {
  float c = fminf(fmaxf(fmaf(y, inv, 12582920.f) - 12582912.f, 0.f), 15.f);
  const float lower = fmaf(c, a, -8.5f * a);
  if (lower > y) c -= 1.f;
  if (lower + a <= y) c += 1.f;
  return __float_as_uint(fminf(fmaxf(c, 0.f), 15.f) + 8388608.f) & 15u;
}
__device__ __forceinline__ uint32_t q4_codes(const float (&x)[8], float d, float inv, bool any_f32) {
  float v[8], c[8];
  const uint64_t magic = f2(12582912.f, 12582912.f), unmagic = f2(-12582912.f, -12582912.f);
  float near = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    f2_get(f2_fma(f2(x[i], x[i + 1]), f2(inv, inv), f2(8.000003814697265625f, 8.000003814697265625f)), v[i], v[i + 1]);
#pragma unroll
    for (int u = 0; u < 2; u++) v[i + u] = fminf(fmaxf(v[i + u], 0.f), 15.f);
    const uint64_t w = f2_add(f2_add(f2(v[i], v[i + 1]), magic), unmagic);
    f2_get(w, c[i], c[i + 1]);
    if (any_f32) near = fminf(near, fminf(v[i] - c[i], v[i + 1] - c[i + 1]));
  }
  if (any_f32 && near < -0.49999f) {
    uint32_t code = 0;
#pragma unroll
    for (int i = 7; i >= 0; i--) code = code << 4 | q4_code(copysignf(1.f, d) * x[i], fabsf(d), fabsf(inv));
    return code;
  }
  const float lo = fmaf(c[3], 4096.f, fmaf(c[2], 256.f, fmaf(c[1], 16.f, c[0] + 8388608.f)));
  const float hi = fmaf(c[7], 4096.f, fmaf(c[6], 256.f, fmaf(c[5], 16.f, c[4] + 8388608.f)));
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
}

// Quantises the eight elements of each lane: a block is four lanes.  Returns the
// lane's codes (element 0 lowest) and the block's scale.  A NaN's bits are the
// largest, so a block that holds one is found by its maximum; its scale is NaN, and
// so is every value that it stands for.  The whole warp calls it.
__device__ __forceinline__ uint32_t q4_block(const float (&x)[8], int lane, bool any_f32, __half* scale) {
  uint32_t top = 0;
  float m = x[0];  // the lane's first element of the lane's largest magnitude
#pragma unroll
  for (int c = 0; c < 8; c++) {
    const uint32_t b = __float_as_uint(x[c]) & 0x7fffffffu;
    if (b > top) {
      top = b;
      m = x[c];
    }
  }
  uint32_t all = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  all = max(all, __shfl_xor_sync(0xffffffffu, all, 2));
  const uint32_t same = __ballot_sync(0xffffffffu, top == all);
  const int first = (lane & 28) + __ffs((same >> (lane & 28)) & 0xfu) - 1;
  m = __shfl_sync(0xffffffffu, m, first);
  // (the limits alone would make a NaN the lower one)
  const __half d = __float2half_rn(all > 0x7f800000u ? m : fminf(fmaxf(m * -0.125f, -65504.f), 65504.f));
  *scale = d;
  const float df = __half2float(d);
  if (!(fabsf(df) > 0.f)) return 0x88888888u;  // zero or NaN
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(df));
  return q4_codes(x, df, inv, any_f32);
}

constexpr int kAppendBlocks = 4;  // per SM: 64 registers hold a row without spills (3: 69 us, 5: 86)

template <typename T, int DH>
__global__ void __launch_bounds__(256, kAppendBlocks) rope_append_kernel(const AppendArgs a) {
  constexpr int LPR = DH / 8, RPB = 256 / LPR, NB = DH / 32;  // lanes per row, rows per pass of the block
  const int lane = threadIdx.x & 31, l = threadIdx.x % LPR, stride = gridDim.x;
  int i = blockIdx.x;
  long long slot = a.slots[i];
  int pos = a.half ? a.positions[i] : 0;
  for (; i < a.n; i += stride) {
    // The block's next token: its slot and position are under way, its rows go into L2.
    const long long here = slot;
    const int at_pos = pos;
    if (i + stride < a.n) {
      slot = a.slots[i + stride];
      if (a.half) pos = a.positions[i + stride];
      constexpr int LINES = DH * (int)sizeof(T) / 128;  // of a row
      for (int r = threadIdx.x; r < (a.H + 2 * a.kv.KV) * LINES; r += 256) {
        const int row = r / LINES - a.H;
        const char* base = reinterpret_cast<const char*>(
            row < 0 ? static_cast<const T*>(a.q) + (i + stride) * a.q_stride
                    : row < a.kv.KV ? static_cast<const T*>(a.k) + (i + stride) * a.k_stride : static_cast<const T*>(a.v) + (i + stride) * a.v_stride);
        const int in = row < 0 ? r : r - (a.H + (row < a.kv.KV ? 0 : a.kv.KV)) * LINES;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(base + in * 128));
      }
    }
    if (here < 0) continue;
    if (here >= a.n_slots || (a.half && (at_pos < 0 || at_pos >= a.table_rows))) {
      if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
      continue;
    }
    // The lane's elements 8l .. 8l + 7 in two groups of four, which may lie on different sides of the pairs' halves.
    float cs[2][4], sn[2][4];  // sn: negative for the lower half of the pairs
    int partner[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int e = 8 * l + 4 * u;
      partner[u] = -1;
#pragma unroll
      for (int c = 0; c < 4; c++) cs[u][c] = 1.f, sn[u][c] = 0.f;
      if (e < 2 * a.half) {
        const bool low = e < a.half;
        const int at = low ? e : e - a.half;
        load4(a.cos_tab + (long long)at_pos * a.half + at, cs[u]);
        load4(a.sin_tab + (long long)at_pos * a.half + at, sn[u]);
        if (low)
#pragma unroll
          for (int c = 0; c < 4; c++) sn[u][c] = -sn[u][c];
        partner[u] = low ? e + a.half : e - a.half;
      }
    }
    // Reads a row's eight elements and their partners (from memory again: the row is in L1).
    auto read = [&](const T* src, float (&x)[8], float (&w)[8]) {
      load8(src + 8 * l, x);
      if (a.half % 8 == 0) {
        if (partner[0] >= 0) load8(src + partner[0], w);
      } else {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float y[4] = {};
          if (partner[u] >= 0) load4(src + partner[u], y);
#pragma unroll
          for (int c = 0; c < 4; c++) w[4 * u + c] = y[c];
        }
      }
    };
    const int sub = threadIdx.x / LPR, first = blockIdx.y * RPB, step = gridDim.y * RPB;  // warp-uniform loops
    // ---- queries ----
    const T* q = static_cast<const T*>(a.q) + i * a.q_stride;
    T* q_out = static_cast<T*>(a.q_out) + (long long)i * a.H * DH + 8 * l;
#pragma unroll 2
    for (int base = first; base < a.H; base += step) {
      const int h = base + sub;
      float x[8], w[8] = {};
      if (h < a.H) read(q + h * DH, x, w);
      __syncwarp();  // in place: a row has been read before any lane writes
      if (h < a.H) {
#pragma unroll
        for (int c = 0; c < 8; c++)
          if (partner[c >> 2] >= 0) x[c] = fmaf(x[c], cs[c >> 2][c & 3], w[c] * sn[c >> 2][c & 3]);
        store8(q_out + h * DH, x);
      }
    }
    // ---- keys and values: the passes go on where the queries' ended, so that a block per pass (few tokens) shares them ----
    const long long at0 = paged_row(a.kv, here >> a.kv.page_log2, 0, (int)(here & ((1 << a.kv.page_log2) - 1)));
    const T* k = static_cast<const T*>(a.k) + i * a.k_stride;
    const T* v = static_cast<const T*>(a.v) + i * a.v_stride;
    const int q_passes = (a.H + RPB - 1) / RPB, begin = (blockIdx.y + gridDim.y - q_passes % gridDim.y) % gridDim.y;
    const int b = l >> 2, t = l & 3;  // block, quarter of it
#pragma unroll 1
    for (int base = begin * RPB; base < 2 * a.kv.KV; base += step) {
      const int r = base + sub;
      const bool row = r < 2 * a.kv.KV, key = r < a.kv.KV;
      const int g = key ? r : r - a.kv.KV;
      float x[8] = {}, w[8] = {};
      if (row && key) read(k + g * DH, x, w);
      if (row && !key) load8(v + g * DH + 8 * l, x);
      __syncwarp();
      const bool turned = __any_sync(0xffffffffu, row && key);
      if (turned) {  // a branch of the warp's: it would pay for f64 instructions that its lanes skip
        if (row && key) {
#pragma unroll
          for (int c = 0; c < 8; c++)  // the products of two f32 values are exact in f64
            if (partner[c >> 2] >= 0)
              x[c] = (float)__dadd_rn(__dmul_rn(x[c], cs[c >> 2][c & 3]), __dmul_rn(w[c], sn[c >> 2][c & 3]));
          if (a.k_out) store8(static_cast<T*>(a.k_out) + ((long long)i * a.kv.KV + g) * DH + 8 * l, x);
        }
      }
      __half d;
      const uint32_t code = q4_block(x, lane, sizeof(T) == 4 || (a.half && turned), &d);
      if (!row) continue;
      const long long at = at0 + ((long long)g << a.kv.page_log2);
      if (key) {
        *reinterpret_cast<uint32_t*>(a.kv.k + at * (DH / 2) + (t * NB + b) * 4) = code;
        if (t == 0) a.kv.ks[at * NB + b] = d;
      } else {
        uint8_t* dst = a.kv.v + at * (DH / 2);
        *reinterpret_cast<uint16_t*>(dst + (2 * t * NB + b) * 2) = (uint16_t)code;
        *reinterpret_cast<uint16_t*>(dst + ((2 * t + 1) * NB + b) * 2) = (uint16_t)(code >> 16);
        if (t == 0) a.kv.vs[at * NB + b] = d;
      }
    }
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

// The values of N codes (lowest bits first) with scale d.
template <int N>
__device__ __forceinline__ void q4_values(uint32_t codes, float d, float (&x)[N]) {
#pragma unroll
  for (int c = 0; c < N; c++) x[c] = (float)((int)((codes >> (4 * c)) & 15u) - 8) * d;
}

template <typename T, int DH>
__global__ void __launch_bounds__(256) read_paged_kernel(const ReadArgs a) {
  constexpr int NB = DH / 32, LPR = DH / 16, RPW = 32 / LPR, UNROLL = 2;  // lanes per row, rows per pass of a warp
  const int lane = threadIdx.x & 31, l = lane % LPR;
  const long long rows = (long long)a.n * a.kv.KV;
  const long long row0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * (RPW * UNROLL) + lane / LPR;
  uint2 kc[UNROLL], vc[UNROLL];
  uint32_t kd[UNROLL];
  uint2 vd[UNROLL];
  bool there[UNROLL];
  const int kb = 2 * l % NB, kt = 2 * l / NB;  // key words 2l, 2l + 1: dimensions 8 kt .. of blocks kb, kb + 1
  const int vb = 4 * l % NB, vg = 4 * l / NB;  // value halfwords 4l .. 4l + 3: dimensions 4 vg .. of blocks vb .. vb + 3
#pragma unroll
  for (int u = 0; u < UNROLL; u++) {
    const long long row = row0 + u * RPW;
    there[u] = false;
    if (row < rows) {
      const int i = (int)(row / a.kv.KV), g = (int)(row - (long long)i * a.kv.KV);
      const long long slot = a.slots[i];
      if (slot >= a.n_slots) {
        if (l == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
      } else if (slot >= 0) {
        const long long at = paged_row(a.kv, slot >> a.kv.page_log2, g, (int)(slot & ((1 << a.kv.page_log2) - 1)));
        kc[u] = *reinterpret_cast<const uint2*>(a.kv.k + at * (DH / 2) + 8 * l);
        vc[u] = *reinterpret_cast<const uint2*>(a.kv.v + at * (DH / 2) + 8 * l);
        kd[u] = *reinterpret_cast<const uint32_t*>(a.kv.ks + at * NB + kb);
        vd[u] = *reinterpret_cast<const uint2*>(a.kv.vs + at * NB + vb);
        there[u] = true;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; u++) {
    if (!there[u]) continue;
    const long long out = (row0 + u * RPW) * DH;
    T* k = static_cast<T*>(a.k_out) + out;
    T* v = static_cast<T*>(a.v_out) + out;
    const float2 ds = f16x2_to_f2(kd[u]), d0 = f16x2_to_f2(vd[u].x), d1 = f16x2_to_f2(vd[u].y);
    float x[8], y[4];
    q4_values(kc[u].x, ds.x, x);
    store8(k + 32 * kb + 8 * kt, x);
    q4_values(kc[u].y, ds.y, x);
    store8(k + 32 * (kb + 1) + 8 * kt, x);
    q4_values(vc[u].x, d0.x, y);
    store4(v + 32 * vb + 4 * vg, y);
    q4_values(vc[u].x >> 16, d0.y, y);
    store4(v + 32 * (vb + 1) + 4 * vg, y);
    q4_values(vc[u].y, d1.x, y);
    store4(v + 32 * (vb + 2) + 4 * vg, y);
    q4_values(vc[u].y >> 16, d1.y, y);
    store4(v + 32 * (vb + 3) + 4 * vg, y);
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
  // Few tokens: a block per pass of rows.  Many: one per token, which walks its rows.
  const int rpb = 256 / (dh / 8), passes = (a.H + rpb - 1) / rpb + (2 * a.kv.KV + rpb - 1) / rpb;
  const bool few = a.n < 4 * h->sm_count;
  const dim3 grid((unsigned)(few ? a.n : std::min(a.n, kAppendBlocks * h->sm_count)), few ? (unsigned)std::min(passes, 65535) : 1u);
  if (dh == 128) rope_append_kernel<T, 128><<<grid, 256, 0, h->stream>>>(a);
  else rope_append_kernel<T, 256><<<grid, 256, 0, h->stream>>>(a);
  return after_launch("hcu_rope_append_paged: launch");
}

template <typename T>
int launch_read(hcu_context* h, const ReadArgs& a, int dh) {
  const int per_block = 8 * 2 * (32 / (dh / 16));  // rows
  const long long blocks = ((long long)a.n * a.kv.KV + per_block - 1) / per_block;
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
  if (p->n > 0x40000000u || p->H > 65535u) return fail(HCU_EINVAL, "%s: n or H too large", op);
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
  if (qs % 8 || ks % 8 || vs % 8) return fail(HCU_EINVAL, "%s: row strides must be multiples of 8 elements", op);
  if (qs < (uint64_t)p->H * kv->Dh || ks < (uint64_t)kv->KV * kv->Dh || vs < (uint64_t)kv->KV * kv->Dh)
    return fail(HCU_EINVAL, "%s: a row stride is shorter than its row", op);
  if ((qs | ks | vs) >> 40) return fail(HCU_EINVAL, "%s: a row stride is too large", op);
  const uintptr_t rows = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         reinterpret_cast<uintptr_t>(k_out) |
                         (p->H ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0);
  if (rows % 16) return fail(HCU_EINVAL, "%s: rows must be 16-byte aligned", op);
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
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16)
    return fail(HCU_EINVAL, "%s: outputs must be 16-byte aligned", op);
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
