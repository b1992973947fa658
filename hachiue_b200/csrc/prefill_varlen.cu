// prefill_varlen.cu - causal attention over packed prompts of different
// lengths (hcu_prefill_varlen).
//
// One warp per (query row, head): lane l holds elements 4l .. 4l + 3, the
// warp walks the query's keys with the online softmax in the log2 domain.
#include "paged.cuh"

namespace hcu {
namespace {

struct VarlenArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* cu_q;
  const int32_t* cu_k;
  long long q_stride, k_stride, v_stride;
  int batch, H, KV, G, window, total_q, total_k;
  float scale_log2;
  uint32_t* status;
};

template <typename T>
__global__ void __launch_bounds__(256) prefill_varlen_kernel(const VarlenArgs a) {
  const int lane = threadIdx.x & 31, h = blockIdx.y, kvh = h / a.G;
  const int b = blockIdx.z;
  const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  if (q0 < 0 || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) {
    if (threadIdx.x == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
    return;
  }
  for (int i = q0 + blockIdx.x * 8 + (threadIdx.x >> 5); i < q1; i += gridDim.x * 8) {
    const int pos = (k1 - k0) - (q1 - q0) + (i - q0);
    const int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    float q[4], acc[4] = {}, m = -INFINITY, l = 0.f;
    load4(static_cast<const T*>(a.q) + (long long)i * a.q_stride + h * 128 + 4 * lane, q);
    for (int t = lo; t <= pos; t++) {
      float k[4], v[4];
      load4(static_cast<const T*>(a.k) + (long long)(k0 + t) * a.k_stride + kvh * 128 + 4 * lane, k);
      load4(static_cast<const T*>(a.v) + (long long)(k0 + t) * a.v_stride + kvh * 128 + 4 * lane, v);
      float x = fmaf(q[0], k[0], fmaf(q[1], k[1], fmaf(q[2], k[2], q[3] * k[3])));
      x = warp_sum(x) * a.scale_log2;
      const float mn = fmaxf(m, x), f = exp2f(m - mn), p = exp2f(x - mn);
      m = mn;
      l = fmaf(l, f, p);
#pragma unroll
      for (int c = 0; c < 4; c++) acc[c] = fmaf(acc[c], f, p * v[c]);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;  // a query that sees no key gives zeros
#pragma unroll
    for (int c = 0; c < 4; c++) acc[c] *= inv;
    store4(static_cast<T*>(a.out) + ((long long)i * a.H + h) * 128 + 4 * lane, acc);
  }
}

}  // namespace
}  // namespace hcu

using hcu::fail;

extern "C" int hcu_prefill_varlen(hcu_handle h, const hcu_prefill_varlen_params* p, const void* q, const void* k,
                                  const void* v, void* out) {
  const char* op = "hcu_prefill_varlen";
  hcu::DeviceScope scope;
  HCU_TRY(hcu::begin_op(h, op));
  if (!p) return fail(HCU_EINVAL, "%s: null params", op);
  if (p->dtype != HCU_DT_BF16 && p->dtype != HCU_DT_F16)
    return fail(HCU_EINVAL, "%s: dtype must be HCU_DT_BF16 or HCU_DT_F16", op);
  if (p->D != 128) return fail(HCU_EUNSUPPORTED, "%s: D=%u (built: 128)", op, p->D);
  if (p->KV == 0 || p->H == 0 || p->H % p->KV)
    return fail(HCU_EINVAL, "%s: H (%u) is not a positive multiple of KV (%u)", op, p->H, p->KV);
  if (p->H > 65535u || p->batch > 65535u) return fail(HCU_EINVAL, "%s: H or batch > 65535", op);
  if (p->total_q > 0x7fffff00u || p->total_k > 0x7fffff00u || p->window > 0x7fffffffu)
    return fail(HCU_EINVAL, "%s: total_q, total_k or window too large", op);
  if (p->batch == 0 || p->total_q == 0) return HCU_OK;
  if (!q || !out || !p->cu_q) return fail(HCU_EINVAL, "%s: null argument", op);
  if (p->total_k && (!k || !v)) return fail(HCU_EINVAL, "%s: null k or v", op);
  if (!p->cu_k && p->total_k != p->total_q) return fail(HCU_EINVAL, "%s: without cu_k, total_k must be total_q", op);
  hcu::VarlenArgs a{};
  a.q_stride = (long long)(p->q_row_stride ? p->q_row_stride : (uint64_t)p->H * 128);
  a.k_stride = (long long)(p->k_row_stride ? p->k_row_stride : (uint64_t)p->KV * 128);
  a.v_stride = (long long)(p->v_row_stride ? p->v_row_stride : (uint64_t)p->KV * 128);
  if (a.q_stride % 8 || a.k_stride % 8 || a.v_stride % 8)
    return fail(HCU_EINVAL, "%s: row strides must be multiples of 8 elements", op);
  if (a.q_stride < (long long)p->H * 128 || a.k_stride < (long long)p->KV * 128 || a.v_stride < (long long)p->KV * 128)
    return fail(HCU_EINVAL, "%s: a row stride is shorter than its row", op);
  if ((a.q_stride | a.k_stride | a.v_stride) >> 32) return fail(HCU_EINVAL, "%s: a row stride is too large", op);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) % 16)
    return fail(HCU_EINVAL, "%s: q, k, v and out must be 16-byte aligned", op);
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.cu_q = p->cu_q;
  a.cu_k = p->cu_k ? p->cu_k : p->cu_q;
  a.batch = (int)p->batch;
  a.H = (int)p->H;
  a.KV = (int)p->KV;
  a.G = a.H / a.KV;
  a.window = (int)p->window;
  a.total_q = (int)p->total_q;
  a.total_k = (int)p->total_k;
  a.scale_log2 = hcu::kLog2e / sqrtf(128.f);
  a.status = h->dev_status;
  const unsigned gx = (unsigned)((a.total_q + 7) / 8 < 1024 ? (a.total_q + 7) / 8 : 1024);
  const dim3 grid(gx, (unsigned)a.H, (unsigned)a.batch);
  if (p->dtype == HCU_DT_BF16) hcu::prefill_varlen_kernel<__nv_bfloat16><<<grid, 256, 0, h->stream>>>(a);
  else hcu::prefill_varlen_kernel<__half><<<grid, 256, 0, h->stream>>>(a);
  return hcu::after_launch("hcu_prefill_varlen: launch");
}
