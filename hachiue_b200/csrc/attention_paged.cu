// attention_paged.cu - decode attention over the paged 4-bit cache
// (hcu_attention_paged).
//
// softmax(q . k / sqrt(Dh)) . v over the visible tokens of each sequence, with
// the online softmax in the log2 domain.  One CTA per (KV head, query row,
// sequence): its warps take tokens in turn, lane l holding elements
// 4l .. 4l + 3 of each 128, and join their (max, sum, accumulator) at the end.
#include "paged.cuh"

namespace hcu {
namespace {

struct PagedAttnArgs {
  const void* q;
  void* out;
  PagedKV kv;
  const int32_t* table;
  const int32_t* context;
  int S, H, G, window, max_context, table_stride;
  float scale_log2;  // log2(e) / sqrt(Dh)
  uint32_t* status;
};

constexpr int kWarps = 8;

template <typename T, int DH>
__global__ void __launch_bounds__(32 * kWarps) attn_paged_kernel(const PagedAttnArgs a) {
  constexpr int NJ = DH / 128, NB = DH / 32;
  __shared__ float part[kWarps][DH + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.x, row = blockIdx.y, b = blockIdx.z;
  const int s = row / a.G, h = g * a.G + row % a.G;
  const size_t at = (((size_t)b * a.S + s) * a.H + h) * DH;
  int n = a.context[b];
  if (n > a.max_context) {
    if (threadIdx.x == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
    n = 0;
  }
  const int pos = n - a.S + s;
  const int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
  float q[NJ][4], acc[NJ][4] = {};
#pragma unroll
  for (int j = 0; j < NJ; j++) load4(static_cast<const T*>(a.q) + at + 128 * j + 4 * lane, q[j]);
  float m = -INFINITY, l = 0.f;
  for (int t = lo + warp; t <= pos; t += kWarps) {
    const int page = a.table[(size_t)b * a.table_stride + (t >> a.kv.page_log2)];
    if (page < 0 || page >= a.kv.n_pages) {
      if (lane == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
      continue;
    }
    const long long r = paged_row(a.kv, page, g, t & ((1 << a.kv.page_log2) - 1));
    float x = 0.f, v[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int blk = 4 * j + (lane >> 3), e = lane & 7;
      const uint32_t kc = *reinterpret_cast<const uint16_t*>(a.kv.k + r * (DH / 2) + ((e >> 1) * NB + blk) * 4 + (e & 1) * 2);
      const uint32_t vc = *reinterpret_cast<const uint16_t*>(a.kv.v + r * (DH / 2) + (e * NB + blk) * 2);
      const float kd = __half2float(a.kv.ks[r * NB + blk]), vd = __half2float(a.kv.vs[r * NB + blk]);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        x = fmaf(q[j][c], (float)((int)((kc >> (4 * c)) & 15u) - 8) * kd, x);
        v[j][c] = (float)((int)((vc >> (4 * c)) & 15u) - 8) * vd;
      }
    }
    x = warp_sum(x) * a.scale_log2;
    const float mn = fmaxf(m, x), f = exp2f(m - mn), p = exp2f(x - mn);
    m = mn;
    l = fmaf(l, f, p);
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) acc[j][c] = fmaf(acc[j][c], f, p * v[j][c]);
  }
#pragma unroll
  for (int j = 0; j < NJ; j++)
#pragma unroll
    for (int c = 0; c < 4; c++) part[warp][128 * j + 4 * lane + c] = acc[j][c];
  if (lane == 0) {
    part[warp][DH] = m;
    part[warp][DH + 1] = l;
  }
  __syncthreads();
  if (warp != 0) return;
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; w++) M = fmaxf(M, part[w][DH]);
  float o[NJ][4] = {};
  for (int w = 0; w < kWarps; w++) {
    if (part[w][DH] == -INFINITY) continue;
    const float f = exp2f(part[w][DH] - M);
    L = fmaf(part[w][DH + 1], f, L);
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) o[j][c] = fmaf(part[w][128 * j + 4 * lane + c], f, o[j][c]);
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;  // a query that sees no token gives zeros
#pragma unroll
  for (int j = 0; j < NJ; j++) {
#pragma unroll
    for (int c = 0; c < 4; c++) o[j][c] *= inv;
    store4(static_cast<T*>(a.out) + at + 128 * j + 4 * lane, o[j]);
  }
}

template <typename T>
int launch(hcu_context* h, const PagedAttnArgs& a, int batch, int dh) {
  const dim3 grid(a.kv.KV, a.S * a.G, batch);
  if (dh == 128) attn_paged_kernel<T, 128><<<grid, 32 * kWarps, 0, h->stream>>>(a);
  else attn_paged_kernel<T, 256><<<grid, 32 * kWarps, 0, h->stream>>>(a);
  return after_launch("hcu_attention_paged: launch");
}

}  // namespace
}  // namespace hcu

using hcu::fail;

extern "C" int hcu_attention_paged(hcu_handle h, const hcu_attention_paged_params* p, const void* q,
                                   const hcu_paged_kv* kv, void* out) {
  const char* op = "hcu_attention_paged";
  hcu::DeviceScope scope;
  HCU_TRY(hcu::begin_op(h, op));
  hcu::PagedAttnArgs a{};
  if (!p) return fail(HCU_EINVAL, "%s: null params", op);
  HCU_TRY(hcu::check_paged(op, kv, &a.kv));
  const int eb = hcu::dtype_bytes(p->dtype);
  if (!eb) return fail(HCU_EINVAL, "%s: unknown dtype %u", op, p->dtype);
  if (p->H == 0 || p->H % kv->KV) return fail(HCU_EINVAL, "%s: H (%u) is not a positive multiple of KV (%u)", op, p->H, kv->KV);
  if (p->S == 0) return fail(HCU_EINVAL, "%s: S must be positive", op);
  if (p->batch == 0) return HCU_OK;
  if (p->batch > 65535u) return fail(HCU_EINVAL, "%s: batch > 65535", op);
  if ((uint64_t)p->S * (p->H / kv->KV) > 65535u) return fail(HCU_EINVAL, "%s: S * H / KV > 65535", op);
  if (p->max_context > 0x7fffff00u || p->windowSize > 0x7fffffffu)
    return fail(HCU_EINVAL, "%s: max_context or windowSize too large", op);
  if (!q || !out || !p->block_table || !p->context) return fail(HCU_EINVAL, "%s: null argument", op);
  if ((uint64_t)p->table_stride * kv->page_size < p->max_context)
    return fail(HCU_EINVAL, "%s: table_stride (%u) pages of %u tokens cannot hold max_context (%u)", op, p->table_stride,
                kv->page_size, p->max_context);
  if (p->table_stride > 0x7fffffffu) return fail(HCU_EINVAL, "%s: table_stride too large", op);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16)
    return fail(HCU_EINVAL, "%s: q and out must be 16-byte aligned", op);
  a.q = q;
  a.out = out;
  a.table = p->block_table;
  a.context = p->context;
  a.S = (int)p->S;
  a.H = (int)p->H;
  a.G = (int)(p->H / kv->KV);
  a.window = (int)p->windowSize;
  a.max_context = (int)p->max_context;
  a.table_stride = (int)p->table_stride;
  a.scale_log2 = hcu::kLog2e / sqrtf((float)kv->Dh);
  a.status = h->dev_status;
  switch (p->dtype) {
    case HCU_DT_F32: return hcu::launch<float>(h, a, (int)p->batch, (int)kv->Dh);
    case HCU_DT_F16: return hcu::launch<__half>(h, a, (int)p->batch, (int)kv->Dh);
    default: return hcu::launch<__nv_bfloat16>(h, a, (int)p->batch, (int)kv->Dh);
  }
}
