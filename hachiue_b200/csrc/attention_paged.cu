// attention_paged.cu - decode attention over the paged 4-bit cache
// (hcu_attention_paged).
//
// softmax(q . k / sqrt(Dh)) . v over the visible tokens of each sequence.  A
// cached row of a head is Dh / 2 bytes of codes and Dh / 32 scales for keys and
// values alike, so a call should take as long as HBM needs for them; what
// stands against that is arithmetic per element: every 4-bit code has to become a tensor-core
// operand.  The codes are therefore expanded in registers into the fragments of
// mma.sync.m16n8k16 (f16 operands, f32 sums), which takes 0.6 instructions per
// key and 1.25 per value element and no trip through shared memory; a tcgen05
// operand would have to be written to shared or tensor memory first, for tiles
// of which the few query rows use a sixteenth.
//
//  * Keys: the bits of a code c, masked out of a word in place, are the f16
//    subnormal c * 2^-24 (or 16 c * 2^-24), which multiplies exactly.  A = 16
//    tokens x 16 dimensions, B = the query columns; the offset 8 of the codes is
//    in the accumulators' start, -8 sum(q), and the block's scale multiplies
//    the f32 sum of its 32 dimensions.
//  * Values: A = 16 dimensions x 16 tokens from the codes of two tokens side by
//    side, (0x6400 | c) - 1032 = c - 8 exactly; B = the probabilities times the
//    token's scale of that block.
//  * Query columns: f32 accuracy takes each query (and each weighted
//    probability) as a sum of two f16 numbers in two columns, 22 bits; the rows
//    of one KV head rarely fill the eight columns, so the second one is free
//    for up to four rows.  bf16 calls with more rows use one f16 number, whose
//    rounding (2^-11) stays below the result's own.  Queries are scaled by a power
//    of two per row, so bf16 and f32 exponents fit f16.
//  * Softmax: log2 domain, one pass, per warp.  The reference point M of a row
//    takes in the exponent of the token's largest value scale, so that the
//    weighted probabilities stay within f16's range whatever the scales are; it
//    moves only when one would pass 2^14.
//
// One CTA per (split of the key axis, KV head, block of query rows, sequence);
// its eight warps take chunks of 32 tokens in turn, each with its own ring of
// bulk copies, and never wait for one another until they join their sums.
// Splits are joined by the CTA that draws the last ticket of its unit.
#include <algorithm>

#include "paged.cuh"

namespace hcu {
namespace {

struct PagedAttnArgs {
  const void* q;
  void* out;
  PagedKV kv;
  const int32_t* table;
  const int32_t* context;
  int S, H, G, R, nrb, window, max_context, table_stride;
  int cps;           // chunks of 32 tokens per split
  float scale_log2;  // log2(e) / sqrt(Dh)
  float* part;       // [units, gridDim.x, RB, DH + 2]: sums, M, l
  int* tickets;      // [units], 0 between calls
  uint32_t* status;
  int dtype;
};

constexpr int NW = 8;          // warps of a CTA
constexpr int CHUNK = 32;      // tokens a warp takes at a time
constexpr float kNoM = -1e30f;  // M of a row that has seen no token
constexpr int kMaxPagedSplits = 256;

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Transposes an 8 x 8 matrix of 16-bit elements held one row per four lanes.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// Two codes (one per 16-bit half, in bits 0-3) as f16 code - 8; HIGH: in bits 4-7, as 16 (code - 8).
template <bool HIGH>
__device__ __forceinline__ uint32_t codes_f16(uint32_t z) {
  const uint32_t x = (z & (HIGH ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
  return h2_bits(__hsub2(bits_h2(x), bits_h2(HIGH ? 0x64806480u : 0x64086408u)));
}

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
}

// Four consecutive elements of a query row of either type.
__device__ __forceinline__ void load4_dt(const void* p, size_t at, int dtype, float (&x)[4]) {
  if (dtype == HCU_DT_F32) load4(static_cast<const float*>(p) + at, x);
  else if (dtype == HCU_DT_F16) load4(static_cast<const __half*>(p) + at, x);
  else load4(static_cast<const __nv_bfloat16*>(p) + at, x);
}
__device__ __forceinline__ void store_dt(void* p, size_t at, int dtype, float x) {
  if (dtype == HCU_DT_F32) static_cast<float*>(p)[at] = x;
  else if (dtype == HCU_DT_F16) static_cast<__half*>(p)[at] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(x);
}

constexpr int paged_stage_bytes(int dh) { return CHUNK * (dh + dh / 8); }  // codes and scales, keys and values
constexpr int paged_stages(int dh) { return dh == 128 ? 3 : 2; }
constexpr size_t paged_smem(int dh) { return 128 + (size_t)NW * paged_stages(dh) * (paged_stage_bytes(dh) + 8); }

// TERMS f16 numbers per query, NC groups of eight columns: RB = 8 NC / TERMS rows per CTA.
template <int DH, int TERMS, int NC>
__global__ void __launch_bounds__(32 * NW, (DH == 128 && NC == 1) ? 2 : 1) attn_paged_kernel(const PagedAttnArgs a) {
  constexpr int NB = DH / 32, ST = paged_stages(DH), SB = paged_stage_bytes(DH);
  constexpr int RG = 8 / TERMS, RB = RG * NC;  // rows per column group, per CTA
  constexpr int NR = 2 / TERMS;                // rows per thread and column group
  constexpr int KB = CHUNK * DH / 2, CB = CHUNK * NB * 2;  // bytes of a stage's codes, of its scales
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, b = blockIdx.z / a.nrb, r0 = (int)(blockIdx.z % a.nrb) * RB;
  const int rows = min(RB, a.R - r0);

  int ctx = a.context[b];
  if (ctx > a.max_context || ctx < 0) {
    if (threadIdx.x == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
    ctx = 0;
  }
  // The tokens that some row of this CTA sees, [lo, hi), and those that all see, [lo_all, hi_all).
  const int pos_first = ctx - a.S + r0 / a.G, pos_last = ctx - a.S + (r0 + rows - 1) / a.G;
  const int lo = a.window > 0 ? max(0, pos_first + 1 - a.window) : 0, hi = max(0, pos_last + 1);
  const int lo_all = a.window > 0 ? max(0, pos_last + 1 - a.window) : 0, hi_all = max(0, pos_first + 1);
  const int c_lo = lo / CHUNK, c_hi = lo < hi ? (hi + CHUNK - 1) / CHUNK : c_lo;
  const int nsplit = max(1, (c_hi - c_lo + a.cps - 1) / a.cps);
  const int split = blockIdx.x;
  if (split >= nsplit) return;
  const int c0 = c_lo + split * a.cps, c1 = min(c_hi, c0 + a.cps);

  // ---- this warp's ring ----
  uint8_t* ring = smem + warp * ST * SB;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + NW * ST * SB) + warp * ST;
  if (lane == 0) {
    for (int i = 0; i < ST; i++) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  const int page_mask = (1 << a.kv.page_log2) - 1;
  const int sub_log2 = min(a.kv.page_log2, 5), subs = CHUNK >> sub_log2;  // a chunk is one page's part or two pages
  // Lane 4s + w issues tensor w (key codes, value codes, key scales, value
  // scales) of part s.  Returns which parts hold data: parts without a visible
  // token are not looked up, parts on a bad page are reported and left out.
  const int* table = a.table + (size_t)b * a.table_stride;
  auto page_of = [&](int c) -> int {
    const int s = lane >> 2, t0 = c * CHUNK + (s << sub_log2);
    if (s >= subs || c >= c1 || t0 >= hi || t0 + (1 << sub_log2) <= lo) return -2;
    const int page = table[t0 >> a.kv.page_log2];
    return page >= 0 && page < a.kv.n_pages ? page : -1;
  };
  auto issue = [&](int c, int stage, int page) -> uint32_t {
    if (page == -1) atomicOr(a.status, HCU_DEVERR_BADARG);
    const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
    const uint32_t ok = (have & 1u) | ((have >> 3) & 2u);  // lanes 0 and 4
    if (lane == 0) mbar_arrive_expect_tx(&full[stage], __popc(ok) * ((2 * KB + 2 * CB) / CHUNK << sub_log2));
    __syncwarp();
    if (page >= 0) {
      const int s = lane >> 2, w = lane & 3, t0 = c * CHUNK + (s << sub_log2);
      const long long row = paged_row(a.kv, page, kvh, t0 & page_mask);
      uint8_t* st = ring + stage * SB;
      const uint8_t* src = w == 0 ? a.kv.k : w == 1 ? a.kv.v : reinterpret_cast<const uint8_t*>(w == 2 ? a.kv.ks : a.kv.vs);
      const int rb = w < 2 ? DH / 2 : NB * 2;
      uint8_t* dst = st + (w < 2 ? w * KB : 2 * KB + (w - 2) * CB) + (s << sub_log2) * rb;
      bulk_load(dst, src + row * rb, (uint32_t)(rb << sub_log2), &full[stage]);
    }
    return ok;
  };
  uint32_t have[ST];
  int next_page;
  {
    int pg[ST];
#pragma unroll
    for (int i = 0; i < ST; i++) pg[i] = page_of(c0 + warp + i * NW);
    next_page = page_of(c0 + warp + ST * NW);
#pragma unroll
    for (int i = 0; i < ST; i++) have[i] = issue(c0 + warp + i * NW, i, pg[i]);
  }

  // ---- query columns: column g of group nc is row / term of this lane's B fragments ----
  uint32_t qf[NC][NB][4];
  float cini[NC][NB][2];
  float rs[NC][NR];  // score = rs * accumulated sum, rows of this thread's accumulator columns
#pragma unroll
  for (int nc = 0; nc < NC; nc++) {
    const int r = nc * RG + (TERMS == 2 ? g >> 1 : g);
    const bool there = r < rows;
    const int rr = r0 + (there ? r : 0), s = rr / a.G, h = kvh * a.G + rr % a.G;
    const size_t at = (((size_t)b * a.S + s) * a.H + h) * DH;
    float q[NB][8], top = 0.f;
#pragma unroll
    for (int i = 0; i < NB; i++) {
      float x[4], y[4];
      load4_dt(a.q, at + 32 * i + 8 * t, a.dtype, x);
      load4_dt(a.q, at + 32 * i + 8 * t + 4, a.dtype, y);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        q[i][c] = there ? x[c] : 0.f;
        q[i][c + 4] = there ? y[c] : 0.f;
        top = fmaxf(top, fmaxf(fabsf(q[i][c]), fabsf(q[i][c + 4])));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^sq brings the row's largest magnitude into [2^13, 2^14)
    const int sq = top > 0.f ? min(127, 140 - (int)(__float_as_uint(top) >> 23)) : 0;
    const float up = __uint_as_float((uint32_t)(max(sq, -126) + 127) << 23);
    const float back = ldexpf(a.scale_log2, 24 - max(sq, -126));
#pragma unroll
    for (int i = 0; i < NB; i++) {
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < 4; m++) {
        // register m: dimensions m and m + 4 of the lane's eight; odd m meets codes times 16
        float v[2];
        __half o[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
          v[c] = q[i][m + 4 * c] * up;
          if (TERMS == 2 && (g & 1)) v[c] -= __half2float(__float2half_rn(v[c]));
          o[c] = __float2half_rn((m & 1) ? v[c] * 0.0625f : v[c]);
          sum += __half2float(o[c]) * ((m & 1) ? 16.f : 1.f);
        }
        qf[nc][i][m] = h2_bits(__halves2half2(o[0], o[1]));
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= -8.f * 5.9604644775390625e-08f;  // -8 * 2^-24
      cini[nc][i][0] = __shfl_sync(0xffffffffu, sum, 8 * t);      // column 2t is lane group g = 2t
      cini[nc][i][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);  // column 2t + 1
    }
    rs[nc][0] = __shfl_sync(0xffffffffu, back, 8 * t);
    if (NR == 2) rs[nc][NR - 1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
  }
  // Visible range of this thread's rows, for chunks that not every row sees whole.
  int row_lo[NC][NR], row_hi[NC][NR];
#pragma unroll
  for (int nc = 0; nc < NC; nc++)
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const int rl = nc * RG + t * NR + r, pos = ctx - a.S + (r0 + rl) / a.G;
      row_hi[nc][r] = rl < rows ? pos : -1;
      row_lo[nc][r] = a.window > 0 ? pos + 1 - a.window : 0;
    }

  float O[2 * NB][NC][4] = {};
  float M[NC][NR], L[NC][NR];
#pragma unroll
  for (int nc = 0; nc < NC; nc++)
#pragma unroll
    for (int r = 0; r < NR; r++) M[nc][r] = kNoM, L[nc][r] = 0.f;
  const int tok = (g >> 1) + 4 * (g & 1);  // token of accumulator row g (row g + 8: 8 more)

  bool ok = true;
  int stage = 0;
  uint32_t phase = 0;
  for (int c = c0 + warp; c < c1; c += NW) {
    if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, a.status))) {
      ok = false;
      break;
    }
    const uint8_t* st = ring + stage * SB;
    uint32_t parts = have[0];
#pragma unroll
    for (int i = 1; i < ST; i++) parts = stage == i ? have[i] : parts;
    const int base = c * CHUNK;
    const bool whole = base >= lo_all && base + CHUNK <= hi_all && parts == (subs == 2 ? 3u : 1u);
    // ---- scores of 32 tokens ----
    float x[2][2][NC][NR];     // [16-token step][accumulator row half][..]: score, log2 units
    float vs[2][2][NB], e[2][2];  // value scales of the thread's tokens, exponent of their largest
#pragma unroll
    for (int j = 0; j < 2; j++) {
      uint32_t kw[2][NB];
      float ks[2][NB];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int row = 16 * j + 8 * u + tok;
        lds_words<NB>(st + row * (DH / 2) + t * NB * 4, kw[u]);
        uint32_t sw[NB / 2];
        lds_words<NB / 2>(st + 2 * KB + row * NB * 2, sw);
        uint32_t vw[NB / 2];
        lds_words<NB / 2>(st + 2 * KB + CB + row * NB * 2, vw);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NB / 2; i++) {
          const float2 f = f16x2_to_f2(sw[i]), w = f16x2_to_f2(vw[i]);
          ks[u][2 * i] = f.x, ks[u][2 * i + 1] = f.y;
          vs[j][u][2 * i] = w.x, vs[j][u][2 * i + 1] = w.y;
          const uint32_t ab = vw[i] & 0x7fff7fffu;
          top = max(top, max(ab >> 16, ab & 0xffffu));
        }
        e[j][u] = (float)((int)(top >> 10) - 14);  // every |scale| of the token is below 2^e
      }
#pragma unroll
      for (int nc = 0; nc < NC; nc++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int r = 0; r < NR; r++) x[j][u][nc][r] = 0.f;
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const uint32_t a0[4] = {kw[0][i] & 0x000f000fu, kw[1][i] & 0x000f000fu, kw[0][i] & 0x00f000f0u,
                                kw[1][i] & 0x00f000f0u};
        const uint32_t w0 = kw[0][i] >> 8, w1 = kw[1][i] >> 8;
        const uint32_t a1[4] = {w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u};
#pragma unroll
        for (int nc = 0; nc < NC; nc++) {
          float d[4];
          const float ini[4] = {cini[nc][i][0], cini[nc][i][1], cini[nc][i][0], cini[nc][i][1]};
          mma16816(d, a0, qf[nc][i][0], qf[nc][i][1], ini);
          mma16816(d, a1, qf[nc][i][2], qf[nc][i][3], d);
#pragma unroll
          for (int u = 0; u < 2; u++) {
            if (TERMS == 2) {
              x[j][u][nc][0] = fmaf(ks[u][i], d[2 * u] + d[2 * u + 1], x[j][u][nc][0]);
            } else {
              x[j][u][nc][0] = fmaf(ks[u][i], d[2 * u], x[j][u][nc][0]);
              x[j][u][nc][NR - 1] = fmaf(ks[u][i], d[2 * u + 1], x[j][u][nc][NR - 1]);
            }
          }
        }
      }
#pragma unroll
      for (int nc = 0; nc < NC; nc++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int r = 0; r < NR; r++) x[j][u][nc][r] *= rs[nc][r];
      if (!whole) {
        // Tokens outside a row's range and on missing pages weigh nothing; what their rows hold is not looked at.
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int tk = 16 * j + 8 * u + tok;
          const bool data = (parts >> (subs == 2 ? j : 0)) & 1u;
          bool any = false;
#pragma unroll
          for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int r = 0; r < NR; r++) {
              const bool see = data && base + tk >= row_lo[nc][r] && base + tk <= row_hi[nc][r];
              x[j][u][nc][r] = see ? x[j][u][nc][r] : -INFINITY;
              any = any || see;
            }
          if (!any) {
            e[j][u] = 0.f;
#pragma unroll
            for (int i = 0; i < NB; i++) vs[j][u][i] = 0.f;
          }
        }
      }
    }
    // ---- reference points: move when a weighted probability would pass 2^14 ----
    bool grow = false;
#pragma unroll
    for (int nc = 0; nc < NC; nc++)
#pragma unroll
      for (int r = 0; r < NR; r++) {
        float w = fmaxf(fmaxf(x[0][0][nc][r] + e[0][0], x[0][1][nc][r] + e[0][1]),
                        fmaxf(x[1][0][nc][r] + e[1][0], x[1][1][nc][r] + e[1][1]));
        grow = grow || w > M[nc][r] + 14.f;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nc = 0; nc < NC; nc++) {
        float f[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
          float w = fmaxf(fmaxf(x[0][0][nc][r] + e[0][0], x[0][1][nc][r] + e[0][1]),
                          fmaxf(x[1][0][nc][r] + e[1][0], x[1][1][nc][r] + e[1][1]));
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
          const float m = w > M[nc][r] + 14.f ? w - 4.f : M[nc][r];
          f[r] = exp2f(M[nc][r] - m);
          M[nc][r] = m;
          L[nc][r] *= f[r];
        }
#pragma unroll
        for (int i = 0; i < 2 * NB; i++)
#pragma unroll
          for (int k = 0; k < 4; k++) O[i][nc][k] *= f[NR == 2 ? (k & 1) : 0];
      }
    }
    // ---- weighted probabilities, values ----
#pragma unroll
    for (int j = 0; j < 2; j++) {
      uint32_t pb[NC][NB][2];  // B fragments: tokens in pairs, column g
#pragma unroll
      for (int nc = 0; nc < NC; nc++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float p[NR];
#pragma unroll
          for (int r = 0; r < NR; r++) {
            p[r] = ex2_approx(x[j][u][nc][r] - M[nc][r]);
            L[nc][r] += p[r];
          }
#pragma unroll
          for (int i = 0; i < NB; i++) {
            uint32_t w;
            if (TERMS == 2) {
              const float y = p[0] * vs[j][u][i];
              const float top = __uint_as_float(__float_as_uint(y) & 0xffffe000u);
              w = h2_bits(__floats2half2_rn(top, y - top));
            } else {
              w = h2_bits(__floats2half2_rn(p[0] * vs[j][u][i], p[NR - 1] * vs[j][u][i]));
            }
            pb[nc][i][u] = movmatrix(w);
          }
        }
      uint32_t vw[4][NB / 2];  // tokens t, t + 4, t + 8, t + 12: halfwords of the lane's dimensions
#pragma unroll
      for (int k = 0; k < 4; k++) lds_words<NB / 2>(st + KB + (16 * j + t + 4 * k) * (DH / 2) + g * NB * 2, vw[k]);
#pragma unroll
      for (int i = 0; i < NB; i++) {
        const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
        uint32_t z0 = __byte_perm(vw[0][i / 2], vw[1][i / 2], sel), z1 = __byte_perm(vw[2][i / 2], vw[3][i / 2], sel);
#pragma unroll
        for (int m = 0; m < 2; m++) {
          const uint32_t av[4] = {codes_f16<false>(z0), codes_f16<true>(z0), codes_f16<false>(z1), codes_f16<true>(z1)};
#pragma unroll
          for (int nc = 0; nc < NC; nc++)
            mma16816(O[2 * i + m][nc], av, pb[nc][i][0], pb[nc][i][1], O[2 * i + m][nc]);
          z0 >>= 8, z1 >>= 8;
        }
      }
    }
    // ---- the stage is free: the chunk ST rounds on ----
    __syncwarp();
    const uint32_t got = issue(c + ST * NW, stage, next_page);
#pragma unroll
    for (int i = 0; i < ST; i++) have[i] = stage == i ? got : have[i];
    next_page = page_of(c + (ST + 1) * NW);
    if (++stage == ST) stage = 0, phase ^= 1;
  }
  // Copies still in flight (none hold data after a whole walk; after a wait that gave up they may) land before the
  // ring is reused below.
  for (int i = 0; i < ST; i++) {
    mbar_wait(&full[stage], phase, a.status);
    if (++stage == ST) stage = 0, phase ^= 1;
  }
  ok = __syncthreads_and(ok);

  // ---- join the warps ----
  constexpr int RS = DH + 2;
  float* buf = reinterpret_cast<float*>(smem);  // [NW][RB][RS]
  static_assert((size_t)NW * RB * RS * 4 <= (size_t)NW * ST * SB, "the warps' sums fit the rings");
#pragma unroll
  for (int nc = 0; nc < NC; nc++)
#pragma unroll
    for (int r = 0; r < NR; r++) {
      float l = L[nc][r];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      float* w = buf + (warp * RB + nc * RG + t * NR + r) * RS;
#pragma unroll
      for (int i = 0; i < NB; i++)
#pragma unroll
        for (int m = 0; m < 2; m++) {
          const float* o4 = O[2 * i + m][nc];
          const int d = 32 * i + 4 * g + 2 * m;
          w[d] = TERMS == 2 ? o4[0] + o4[1] : o4[r];
          w[d + 1] = (TERMS == 2 ? o4[2] + o4[3] : o4[2 + r]) * 0.0625f;
        }
      if (g == 0) w[DH] = M[nc][r], w[DH + 1] = l;
    }
  __syncthreads();
  const int unit = ((b * a.kv.KV + kvh) * a.nrb) + (int)(blockIdx.z % a.nrb);
  float* mine = a.part + ((size_t)unit * gridDim.x + split) * RB * RS;
  for (int i = threadIdx.x; i < RB * DH; i += 32 * NW) {
    const int r = i / DH, d = i % DH;
    if (r >= rows) break;
    float m = kNoM;
#pragma unroll
    for (int w = 0; w < NW; w++) m = fmaxf(m, buf[(w * RB + r) * RS + DH]);
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float f = exp2f(buf[(w * RB + r) * RS + DH] - m);
      o = fmaf(buf[(w * RB + r) * RS + d], f, o);
      l = fmaf(buf[(w * RB + r) * RS + DH + 1], f, l);
    }
    if (nsplit == 1) {
      const int rr = r0 + r, s = rr / a.G, h = kvh * a.G + rr % a.G;
      const float y = l > 0.f ? o / l : (l == 0.f ? 0.f : l);  // no token: zeros; NaN stays
      store_dt(a.out, (((size_t)b * a.S + s) * a.H + h) * DH + d, a.dtype, y);
    } else {
      mine[r * RS + d] = o;
      if (d == 0) mine[r * RS + DH] = m, mine[r * RS + DH + 1] = l;
    }
  }
  if (nsplit == 1) return;

  // ---- join the splits: the CTA that draws the unit's last ticket ----
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&a.tickets[unit], 1) == nsplit - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float* all = a.part + (size_t)unit * gridDim.x * RB * RS;
  for (int i = threadIdx.x; i < rows * DH; i += 32 * NW) {
    const int r = i / DH, d = i % DH;
    float m = kNoM, o = 0.f, l = 0.f;
    for (int s = 0; s < nsplit; s++) m = fmaxf(m, __ldcg(all + (size_t)s * RB * RS + r * RS + DH));
    for (int s = 0; s < nsplit; s++) {
      const float* p = all + (size_t)s * RB * RS + r * RS;
      const float f = exp2f(__ldcg(p + DH) - m);
      o = fmaf(__ldcg(p + d), f, o);
      l = fmaf(__ldcg(p + DH + 1), f, l);
    }
    const int rr = r0 + r, s = rr / a.G, h = kvh * a.G + rr % a.G;
    const float y = l > 0.f ? o / l : (l == 0.f ? 0.f : l);
    store_dt(a.out, (((size_t)b * a.S + s) * a.H + h) * DH + d, a.dtype, y);
  }
  if (threadIdx.x == 0) a.tickets[unit] = 0;  // re-armed for the next call
}

template <int DH, int TERMS, int NC>
int launch(hcu_context* h, PagedAttnArgs a, int batch) {
  const char* op = "hcu_attention_paged";
  constexpr int RB = 8 * NC / TERMS;
  constexpr size_t smem = paged_smem(DH);
  auto kern = attn_paged_kernel<DH, TERMS, NC>;
  static std::atomic<uint64_t> attr_done{0};  // per device
  HCU_TRY(once_per_device(attr_done, h->device, [&]() -> int {
    return check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), op);
  }));
  a.nrb = (a.R + RB - 1) / RB;
  const long long units = (long long)batch * a.kv.KV * a.nrb;
  if ((long long)batch * a.nrb > 65535) return fail(HCU_EINVAL, "%s: batch x query row blocks > 65535", op);
  // Keys per split: enough CTAs for several rounds of the GPU, which evens out sequences of different lengths, but no
  // fewer than one round of the warps.
  const int span = a.window > 0 ? (int)std::min<long long>(a.max_context, (long long)a.window + a.S + CHUNK) : a.max_context;
  const int chunks = std::max(1, (span + CHUNK - 1) / CHUNK + 1);
  const long long want = std::max(1LL, (8LL * 2 * h->sm_count + units - 1) / units);
  int cps = (int)std::max<long long>(NW, (chunks + want - 1) / want);
  if (h->opt_attn_chunk > 0) cps = (int)std::max<long long>(1, std::min<long long>((h->opt_attn_chunk + CHUNK - 1) / CHUNK, chunks));
  cps = std::max(cps, (chunks + kMaxPagedSplits - 1) / kMaxPagedSplits);
  int splits = (chunks + cps - 1) / cps;
  const size_t record = (size_t)RB * (DH + 2) * sizeof(float);
  const size_t room = h->workspace_bytes > kTicketBytes ? h->workspace_bytes - kTicketBytes : 0;
  const long long fit = (long long)(room / (record * (size_t)units));
  if (units > kMaxUnits || fit < 2) {
    cps = chunks, splits = 1;  // no room for partial sums: one CTA walks all keys
  } else if (splits > fit) {
    cps = (int)((chunks + fit - 1) / fit);
    splits = (chunks + cps - 1) / cps;
  }
  a.cps = cps;
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(h->workspace) + kTicketBytes);
  a.tickets = static_cast<int*>(h->workspace);
  kern<<<dim3((unsigned)splits, (unsigned)a.kv.KV, (unsigned)(batch * a.nrb)), 32 * NW, smem, h->stream>>>(a);
  return after_launch("hcu_attention_paged: launch");
}

template <int DH>
int launch_dh(hcu_context* h, const PagedAttnArgs& a, int batch) {
  // One f16 number per query where the result is rounded to bf16 anyway and the rows fill more than four columns.
  if (a.R <= 4) return launch<DH, 2, 1>(h, a, batch);
  if (a.dtype == HCU_DT_BF16) return a.R <= 8 ? launch<DH, 1, 1>(h, a, batch) : launch<DH, 1, 2>(h, a, batch);
  return launch<DH, 2, 2>(h, a, batch);
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
  a.window = p->windowSize >= p->max_context ? 0 : (int)p->windowSize;  // a window as long as the longest sequence hides nothing
  a.max_context = (int)p->max_context;
  a.table_stride = (int)p->table_stride;
  a.scale_log2 = hcu::kLog2e / sqrtf((float)kv->Dh);
  a.status = h->dev_status;
  a.R = a.S * a.G;
  a.dtype = (int)p->dtype;
  return kv->Dh == 128 ? hcu::launch_dh<128>(h, a, (int)p->batch) : hcu::launch_dh<256>(h, a, (int)p->batch);
}
