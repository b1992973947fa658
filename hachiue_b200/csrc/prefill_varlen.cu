// prefill_varlen.cu - causal attention over packed prompts of different
// lengths (hcu_prefill_varlen), on tcgen05.
//
// O = softmax(Q K^T / sqrt(D) + mask) V per sequence and head, one pass over
// 128-key tiles with the running maximum and sum of the softmax.  The work is
// 4 D flops per visible (query, key) pair, bound by the tensor pipe and, at the
// same rate, by the exponentials: a 128 x 128 tile takes 1024 cycles of
// tcgen05.mma (two products) and 1024 cycles of the SFU (16 per cycle).
//
//  * Rows: the G query heads of a KV head are packed, row i * G + head, so that
//    a tile of 128 rows covers 128 / G queries: short prompts fill tiles, a
//    diagonal wastes fewer keys, and any G works.  A work item is 256 rows (two
//    tiles) of one sequence and KV head; a small kernel sorts the items by their
//    number of key tiles, so that the persistent CTAs' shares are near equal
//    whatever the lengths are.  (A call with no more items than SMs needs no list.)
//  * Warp roles: K / V by TMA (warp 0), tcgen05.mma of each tile (warps 1, 2: one
//    warp for both spent more time on its barriers than the products take), Q tiles
//    by TMA, or row by row with cp.async where G does not divide 128 (warp 3), and a
//    softmax warpgroup per tile, one thread per row.  S
//    is in TMEM, P goes back over its columns, O stays in TMEM across the keys.
//    While one tile's softmax runs the tensor cores work on the other tile.
//  * O is rescaled only when a row's maximum grows by more than 2^8: P stays
//    below 2^8 otherwise and O / l cancels the stale maximum.
//  * Keys and values behind a sequence's end have no influence: scores are
//    selected, value rows are zeroed in shared memory.  Masked keys inside the sequence
//    meet P = 0; where such a value is not finite the row's result is not either.  A CTA
//    that stored such a row (or one that overflowed: P reaches 2^8, so values of bf16's
//    last 2^9 may) goes over its items once more when all of them are done and no wait
//    is open, and computes again, over their visible keys alone, the rows whose result
//    no visible value explains (mend_rows: slow and exact).
//
// Measured, bf16, D = 128, calls in a row (which run at the power cap): 8192 tokens in
// eight prompts of 1 to 3001, 32 / 8 heads, 162 us, 863 TFLOP/s (0.51 of the library's
// dense burst rate); 32772 tokens, 16 / 4 heads, window 1024, 289 us, 832.  Single calls
// with L2 flushed take 153 and 261.  A pair of tiles takes 3300 cycles, 2900 of them the
// chain S -> softmax -> P -> P V of one row; tensor pipe 59 %, SFU 59 %.
#include <algorithm>

#include "paged.cuh"
#include "tcgen05.cuh"

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
  float scale_log2;  // log2(e) / sqrt(D)
  int* blocks;       // [batch + 1]: blocks of 256 rows before each sequence
  int4* items;       // [2 * blocks]: {first query, queries, first key, keys}, {first packed row, first tile's key, tiles, 0}
  uint32_t recip_G, recip_KV;  // for quot()
  int q_tma;         // G divides 128: a tile's rows are one box of Q
  int direct;        // every CTA has one item at most and finds it itself
  uint32_t* status;
};

constexpr int BM = 128, BN = 128, HD = 128;
constexpr int BOX = BM * 128;  // [128 rows x 64 elements]
constexpr int TILE = 2 * BOX;  // [128 x 128]
constexpr int KV_STAGES = 2, KV_STAGE = 2 * TILE;
constexpr int Q_SLOTS = 3;     // tiles of queries: an item's two and the next one's first
constexpr float RESCALE_LOG2 = 8.f;
constexpr uint32_t REG_CTRL = 56, REG_SOFTMAX = 224;
static_assert(128 * REG_CTRL + 256 * REG_SOFTMAX == 384 * 168, "register split");

// n / d for 0 <= n < 2^31 by the host's recip = min(2^32 - 1, 2^32 / d + 1): the product is off by one at most.
__device__ __forceinline__ int quot(int n, int d, uint32_t recip) {
  int q = (int)__umulhi((uint32_t)n, recip);
  if (q * d > n) q--;
  if (n - q * d >= d) q++;
  return q;
}

// ---- the items, longest first ------------------------------------------------
constexpr int kBins = 1024;

// Key tiles of rows [r0, r1) of a sequence.
__device__ __forceinline__ int2 key_tiles(int r0, int r1, int G, int lq, int lk, int W) {
  const int off = lk - lq, first = off + r0 / G, last = off + min(lq - 1, (r1 - 1) / G);
  const int lo = W > 0 ? max(0, first - W + 1) : 0;
  const int n_first = lo / BN * BN;
  return make_int2(n_first, last < n_first ? 1 : (last - n_first) / BN + 1);
}

// One block: counts the sequences' blocks of 256 rows, sorts them by their number of key tiles (a counting sort, descending)
// and writes them out.  Sequences whose offsets are not in order or not within the tensors are reported and left out; one that
// begins below any offset before it counts as such, so that the others do not overlap and their blocks fit the list.
__global__ void __launch_bounds__(1024) varlen_items_kernel(const VarlenArgs a) {
  __shared__ int bins[kBins], part[32], top_part[32], base, top_base;
  asm volatile("griddepcontrol.launch_dependents;");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  bins[tid] = 0;
  if (tid == 0) base = 0, top_base = 0;
  __syncthreads();
  for (int b0 = 0; b0 < a.batch; b0 += 1024) {
    const int b = b0 + tid;
    // the largest offset up to this sequence's first
    int top = b < a.batch ? a.cu_q[b] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, top, o);
      if (lane >= o) top = max(top, x);
    }
    if (lane == 31) top_part[warp] = top;
    __syncthreads();
    top = max(top, top_base);
    for (int w = 0; w < warp; w++) top = max(top, top_part[w]);
    int n = 0;
    if (b < a.batch) {
      const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
      if (q0 < top || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) atomicOr(a.status, HCU_DEVERR_BADARG);
      else n = (int)(((long long)(q1 - q0) * a.G + 2 * BM - 1) / (2 * BM));
    }
    int pre = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += x;
    }
    if (lane == 31) part[warp] = pre;
    __syncthreads();
    int before = base;
    for (int w = 0; w < warp; w++) before += part[w];
    if (b < a.batch) a.blocks[b] = before + pre - n;
    __syncthreads();
    if (tid == 1023) base = before + pre, top_base = top;
    __syncthreads();
  }
  const int total = base;
  if (tid == 0) a.blocks[a.batch] = total;
  __syncthreads();
  for (int pass = 0; pass < 2; pass++) {
    for (int i = tid; i < total; i += 1024) {
      int lo = 0, hi = a.batch - 1;  // the last sequence whose blocks begin at or before i
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.blocks[mid] <= i) lo = mid;
        else hi = mid - 1;
      }
      const int q0 = a.cu_q[lo], lq = a.cu_q[lo + 1] - q0, k0 = a.cu_k[lo], lk = a.cu_k[lo + 1] - k0, blk = i - a.blocks[lo];
      const int r0 = blk * 2 * BM, rows = (int)min((long long)lq * a.G - r0, 2LL * BM);
      const int2 tiles = key_tiles(r0, r0 + rows, a.G, lq, lk, a.window);
      const int bin = kBins - 1 - min(tiles.y, kBins - 1);
      if (pass == 0) {
        atomicAdd(&bins[bin], 1);
      } else {
        const int at = atomicAdd(&bins[bin], 1);
        a.items[2 * at] = make_int4(q0, lq, k0, lk);
        a.items[2 * at + 1] = make_int4(r0, tiles.x, tiles.y, 0);
      }
    }
    __syncthreads();
    if (pass == 0) {
      const int n = bins[tid];
      int pre = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, pre, o);
        if (lane >= o) pre += x;
      }
      if (lane == 31) part[warp] = pre;
      __syncthreads();
      for (int w = 0; w < warp; w++) pre += part[w];
      bins[tid] = pre - n;
      __syncthreads();
    }
  }
}

// ---- helpers ---------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// max(a, b, c) in one instruction (three-input max.f32, sm_100).
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Scores of columns outside lo..hi (tile columns) become -inf, in one 32-column chunk beginning at column C0: a bit per
// column, tested one by one.  Returns whether no row of the warp keeps any column of it (warp-uniform; the chunk is then left
// as it is and skipped).
template <int C0>
__device__ __forceinline__ bool mask_chunk(uint32_t (&r)[32], int lo, int hi) {
  const int a = min(max(lo - C0, 0), 32), b = min(max(hi + 1 - C0, 0), 32);  // columns a .. b - 1 stay
  const uint32_t keep = (b == 32 ? 0xffffffffu : (1u << b) - 1u) & (a == 32 ? 0u : 0xffffffffu << a);
  if (__all_sync(0xffffffffu, keep == 0xffffffffu)) return false;
  if (__all_sync(0xffffffffu, keep == 0u)) return true;
#pragma unroll
  for (int i = 0; i < 32; i++) r[i] = (keep & (1u << i)) ? r[i] : 0xff800000u;  // -inf
  return false;
}
__device__ __forceinline__ void chunk_max(const uint32_t (&r)[32], float (&mx)[4]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2)
    mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
}

// P of one 32-column chunk as 16 words pk[OFF..], added to the row's sums.
template <bool BF16, int OFF>
__device__ __forceinline__ void chunk_p(const uint32_t (&r)[32], bool empty, uint64_t scale2, uint64_t negm2, uint64_t (&ls2)[2],
                                        uint32_t (&pk)[32]) {
  if (empty) {
#pragma unroll
    for (int i = 0; i < 16; i++) pk[OFF + i] = 0u;
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; i++) {
    float v0, v1;
    f2_get(f2_fma(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), scale2, negm2), v0, v1);
    const float p0 = ex2_approx(v0), p1 = ex2_approx(v1);
    ls2[i & 1] = f2_add(ls2[i & 1], f2(p0, p1));
    pk[OFF + i] = pack16<BF16>(p0, p1);
  }
}

// Barriers by their 32-bit shared-memory address (generic pointers to a dozen of them cost the issuing warp its registers).
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_try_sleep(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}
// Bounded wait of a whole warp (true on every lane or on none): the MMA warp polls, the others sleep and leave it the
// issue slots.
template <bool POLL>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t* status) {
  bool ok = bar_try(bar, parity);
  if (!ok) {
    const uint64_t t0 = globaltimer();
    for (uint32_t n = 1; !(ok = POLL ? bar_try(bar, parity) : bar_try_sleep(bar, parity)); n++) {
      if ((!POLL || (n & 63) == 0) && globaltimer() - t0 > HCU_WAIT_NS) {
        if (status) atomicOr(status, HCU_DEVERR_TIMEOUT);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Barriers of a CTA, in order.
enum Bar { kQFull = 0, kQEmpty = 3, kKFull = 6, kKEmpty = 8, kVFull = 10, kVEmpty = 12, kSFull = 14, kPVDone = 16, kPHalf = 18, kPFull = 20,
           kOFree = 22, kSRead = 24, kBars = 26 };

// A work item: 256 packed rows of one sequence and KV head.  A role loads an item's words while it works on the item
// before and unpacks them when it gets there.
struct RawItem {
  int4 x, y;
  int g;  // KV head; -1: no item
};
struct Item {
  int q0, lq, k0, lk, g, r0;  // first query and their number, first key and their number, KV head, first packed row
  int n_first, ntiles;        // first key of the first tile, tiles of the item
};
__device__ __forceinline__ Item unpack(const RawItem& r) {
  return Item{r.x.x, r.x.y, r.x.z, r.x.w, r.g, r.y.x, r.y.y, r.y.z};
}

// The k-th item of this CTA: rounds of gridDim.x items, forwards in even rounds and backwards in odd ones (costs fall
// with the index).
__device__ __forceinline__ int item_index(int k) {
  const int P = (int)gridDim.x, c = (int)blockIdx.x;
  return k * P + ((k & 1) ? P - 1 - c : c);
}

// The item of this CTA where there are no more items than CTAs: each thread takes a sequence (at most kDirectBatch), checks it
// as varlen_items_kernel does, and the one whose blocks hold the CTA's writes the item.  A launch less: 77 tokens of
// 16 / 8 heads take 8.3 us in a replayed graph, through the list 10.0.
constexpr int kDirectBatch = 384;
__device__ __noinline__ void own_item(const VarlenArgs& a, RawItem* item, int* scan) {
  const int b = threadIdx.x, lane = b & 31, warp = b >> 5;
  int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
  if (b < a.batch) q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  int top = q0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, top, o);
    if (lane >= o) top = max(top, x);
  }
  if (lane == 31) scan[warp] = top;
  if (b == 0) item->g = -1;
  __syncthreads();
  top = max(top, 0);
  for (int w = 0; w < warp; w++) top = max(top, scan[w]);
  int n = 0;
  if (b < a.batch) {
    if (q0 < top || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) {
      if (blockIdx.x == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
    } else {
      n = (int)(((long long)(q1 - q0) * a.G + 2 * BM - 1) / (2 * BM));
    }
  }
  int pre = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, pre, o);
    if (lane >= o) pre += x;
  }
  if (lane == 31) scan[12 + warp] = pre;
  __syncthreads();
  for (int w = 0; w < warp; w++) pre += scan[12 + w];
  const int e = blockIdx.x / a.KV;
  if (e >= pre - n && e < pre) {
    const int lq = q1 - q0, lk = k1 - k0, r0 = (e - (pre - n)) * 2 * BM, rows = (int)min((long long)lq * a.G - r0, 2LL * BM);
    const int2 tiles = key_tiles(r0, r0 + rows, a.G, lq, lk, a.window);
    item->x = make_int4(q0, lq, k0, lk);
    item->y = make_int4(r0, tiles.x, tiles.y, 0);
    item->g = blockIdx.x % a.KV;
  }
}

// ---- rows to be computed again -------------------------------------------------
struct Mend {
  int any;             // a row of the half was stored with a result that is not finite
  int late;            // a wait of the half ran out: its results are not all there
  int rows[4];         // per warp: some row of the present item's is one
  // Dimensions, a bit each.  need: of such results, the infinite ones (words 0 .. 3) and the NaN ones (4 .. 7).  seen: where a
  // value that every row of the half sees is infinite or NaN (0 .. 3), is NaN (4 .. 7).
  uint32_t need[8], seen[8];
};
constexpr uint32_t kNoSum = 0xffffffffu;  // a stored row without a sum (NaN, infinite or zero): NaN for good (no conversion gives this one)

// Two elements: bits 0, 1 infinite or NaN; bits 4, 5 NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  const uint32_t a = w & 0x7fffu, b = w >> 16 & 0x7fffu;
  return (a >= E ? 1u : 0u) | (b >= E ? 2u : 0u) | (a > E ? 16u : 0u) | (b > E ? 32u : 0u);
}
// Four: bits 0 .. 3 and 4 .. 7.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite4(uint2 w) { return not_finite<BF16>(w.x) | not_finite<BF16>(w.y) << 2; }

__device__ __forceinline__ void half_sync(int hd) { asm volatile("bar.sync %0, 128;" ::"r"(1 + hd) : "memory"); }

// One row over its visible keys lo .. hi, by a warp: a lane's keys are lo + lane, 32 apart.  Two passes, so that the weights are
// divided by their sum before they meet the values.
template <bool BF16>
__device__ __noinline__ void row_alone(const VarlenArgs& a, int q_row, int head, int k0, int lo, int hi) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const int lane = threadIdx.x & 31, g = head / a.G;
  const T* q = static_cast<const T*>(a.q) + (long long)q_row * a.q_stride + head * HD;
  const T* k = static_cast<const T*>(a.k) + (long long)k0 * a.k_stride + g * HD;
  const T* v = static_cast<const T*>(a.v) + (long long)k0 * a.v_stride + g * HD;
  auto score = [&](int t) {
    float x = 0.f;
#pragma unroll 8
    for (int d = 0; d < HD; d += 8) {
      float y[8], z[8];
      load8(q + d, y);
      load8(k + (long long)t * a.k_stride + d, z);
#pragma unroll
      for (int c = 0; c < 8; c++) x = fmaf(y[c], z[c], x);
    }
    return x * a.scale_log2;
  };
  float m = -INFINITY, l = 0.f;
  for (int t = lo + lane; t <= hi; t += 32) {
    const float x = score(t), mn = fmaxf(m, x);
    if (x == -INFINITY) continue;  // no weight
    l = fmaf(l, exp2f(m - mn), exp2f(x - mn));
    m = mn;
  }
  const float top = warp_max(m);
  l = warp_sum(m == -INFINITY ? l : l * exp2f(m - top));
  const float inv = 1.f / l;
  float acc[4] = {};
  for (int t0 = lo; t0 <= hi; t0 += 32) {
    const float p = t0 + lane <= hi ? exp2f(score(t0 + lane) - top) * inv : 0.f;
    for (int j0 = 0; j0 < min(32, hi - t0 + 1); j0 += 8) {
      float y[8][4];
#pragma unroll
      for (int j = 0; j < 8; j++) load4(v + (long long)min(t0 + j0 + j, hi) * a.v_stride + 4 * lane, y[j]);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float w = __shfl_sync(0xffffffffu, p, j0 + j);
        if (t0 + j0 + j <= hi)
#pragma unroll
          for (int c = 0; c < 4; c++) acc[c] = fmaf(w, y[j][c], acc[c]);
      }
    }
  }
  store4(static_cast<T*>(a.out) + ((long long)q_row * a.H + head) * HD + 4 * lane, acc);
}

// Of a half's 128 rows of an item, computes those again whose stored result the values that they see do not explain.  An
// infinity is explained by a visible value that is not finite, a NaN by a visible NaN, or by a visible infinity where no
// hidden value of the item's tiles is not finite.  By the half's four warps; `tid` 0 .. 127 is also the row.
template <bool BF16>
__device__ __noinline__ void mend_rows(const VarlenArgs& a, const Item it, int hd, int tid, Mend& s) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const int lane = tid & 31, warp = tid >> 5, off = it.lk - it.lq;
  const int first = it.r0 + hd * BM, r = first + tid, qi = r / a.G, head = it.g * a.G + r % a.G;
  const int q_last = min(it.lq - 1, (first + BM - 1) / a.G);
  auto first_key = [&](int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; };
  uint32_t bad[8] = {};  // this thread's row: dimensions, as in Mend::need
  if (qi < it.lq && off + qi >= 0) {
    const uint4* row = reinterpret_cast<const uint4*>(static_cast<const T*>(a.out) + ((long long)(it.q0 + qi) * a.H + head) * HD);
    if (row->x != kNoSum)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const uint4 w = row[i];
        const uint32_t f = not_finite4<BF16>(make_uint2(w.x, w.y)), h = not_finite4<BF16>(make_uint2(w.z, w.w));
        const uint32_t inf = (f & 15u) | (h & 15u) << 4, nan = f >> 4 | h & 0xf0u;
        bad[i / 4] |= (inf & ~nan) << (8 * (i & 3));
        bad[4 + i / 4] |= nan << (8 * (i & 3));
      }
  }
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) any |= bad[i];
  if (tid < 8) s.need[tid] = s.seen[tid] = 0u;
  half_sync(hd);
  if (any)
#pragma unroll
    for (int i = 0; i < 8; i++) atomicOr(&s.need[i], bad[i]);
  const bool some = __any_sync(0xffffffffu, any != 0);
  if (lane == 0) s.rows[warp] = some;
  half_sync(hd);
  if (!(s.rows[0] | s.rows[1] | s.rows[2] | s.rows[3])) return;
  // A lane has dimensions 4 lane .. + 3: bits 0 .. 3 and 4 .. 7 of these masks are words 0 .. 3 and 4 .. 7 of Mend's.
  const int word = lane >> 3, bit = 4 * (lane & 7);
  auto part = [&](const uint32_t* w) { return (w[word] >> bit & 15u) | (w[4 + word] >> bit & 15u) << 4; };
  const T* v = static_cast<const T*>(a.v) + (long long)it.k0 * a.v_stride + it.g * HD + 4 * lane;
  auto value = [&](int t) { return not_finite4<BF16>(*reinterpret_cast<const uint2*>(v + (long long)t * a.v_stride)); };
  // Keys that every row of the half sees: a warp looks at eight of every 32.
  const int all_lo = first_key(off + q_last), all_hi = off + first / a.G;
  const uint32_t mine = part(s.need), dims = (mine | mine >> 4) & 15u;
  for (int t0 = all_lo + 8 * warp; t0 <= all_hi; t0 += 32) {
    uint32_t f = 0;
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (t0 + j <= all_hi) f |= value(t0 + j);
    if (f &= dims * 17u) {
      atomicOr(&s.seen[word], (f & 15u) << bit);
      atomicOr(&s.seen[4 + word], (f >> 4) << bit);
    }
    const volatile uint32_t* now = s.seen;
    if (__all_sync(0xffffffffu, (mine & ~((now[word] >> bit & 15u) | (now[4 + word] >> bit & 15u) << 4)) == 0)) break;
  }
  half_sync(hd);
  const uint32_t seen = part(s.seen);
  uint32_t left = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) left |= bad[i] & ~s.seen[i];
  for (uint32_t rows = __ballot_sync(0xffffffffu, left != 0); rows; rows &= rows - 1) {
    const int src = __ffs(rows) - 1;
    const int pos = __shfl_sync(0xffffffffu, off + qi, src), h = __shfl_sync(0xffffffffu, head, src), lo = first_key(pos);
    uint32_t open = 0;  // of this lane's four dimensions
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t w = __shfl_sync(0xffffffffu, bad[i], src);
      if ((i & 3) == word) open |= (w >> bit & 15u) << (i & 4);
    }
    // the keys that this row sees and some other of the half does not
    uint32_t visible = seen;
    for (int t = lo; t < min(all_lo, pos + 1); t++) visible |= value(t);
    for (int t = max(max(lo, all_lo), all_hi + 1); t <= pos; t++) visible |= value(t);
    open &= ~visible;
    if (const uint32_t either = open >> 4 & visible & 15u; __any_sync(0xffffffffu, either != 0)) {
      uint32_t hidden = 0;
      for (int t = it.n_first; t < lo; t++) hidden |= value(t);
      for (int t = pos + 1; t < min(it.lk, it.n_first + it.ntiles * BN); t++) hidden |= value(t);
      open &= ~((either & ~hidden) << 4);
    }
    if (__any_sync(0xffffffffu, open != 0)) row_alone<BF16>(a, it.q0 + pos - off, h, it.k0, lo, pos);
  }
  half_sync(hd);  // the masks are free again
}

// TMEM (512 columns): O of the two halves, P of the two, and ONE buffer for S.
// A softmax thread takes its whole row of S into registers at once, so the
// buffer is free again some 100 cycles after the product is done, and the
// halves share it in turn: the next scores of a half are computed while it
// still works on the ones before.  (With a buffer each and P written over S a
// half's products and its softmax took turns: 1500 of 4200 cycles per tile.)
constexpr uint32_t kColP = 256, kColS = 384;

// Barriers run on across items; every role advances the same counters.  Tile t
// is the t-th key tile of this CTA's items; each half takes every tile.
//   q_full / q_empty          per query tile (slot = tiles so far mod 3),
//   k_full .. v_empty         per tile (rings of two; each half releases every tile),
//   s_full, p_half, p_full    per tile and half,
//   pv_done                   per tile and half: P has been read, O is whole,
//   s_read                    per tile and half: S is in registers (the buffer is the other half's),
//   o_free                    per item and half: O has been read, the next P.V may overwrite it.
template <bool BF16>
__global__ void __launch_bounds__(384, 1)
    prefill_varlen_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const __grid_constant__ VarlenArgs a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qsm = smem;                    // [Q_SLOTS][TILE]
  uint8_t* kvsm = qsm + Q_SLOTS * TILE;   // [KV_STAGES][K tile | V tile]
  __shared__ uint64_t bars[kBars];
  __shared__ uint32_t tmem_slot;
  __shared__ RawItem s_item;
  __shared__ int s_scan[24];
  __shared__ Mend s_mend[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid < 2) s_mend[tid].any = s_mend[tid].late = 0;
  if (tid == 0) {
    for (int i = 0; i < kBars; i++)
      mbar_init(&bars[i], i >= kPHalf ? 4 : (i >= kKEmpty && i < kVFull) || (i >= kVEmpty && i < kSFull) ? 2 : 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  if (a.direct) own_item(a, &s_item, s_scan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8 * i; };
  auto wait = [&](int i, uint32_t parity) { return bar_wait<false>(bar0 + 8 * i, parity, a.status); };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_items = a.direct ? 0 : a.blocks[a.batch] * a.KV;
  auto load_item = [&](int k) {
    const int idx = item_index(k);
    RawItem r{make_int4(0, 0, 0, 0), make_int4(0, 0, 0, 0), -1};
    if (a.direct && k == 0) {
      r.g = s_item.g;
      r.x = s_item.x;
      r.y = s_item.y;
    }
    if (idx < n_items) {
      const int e = quot(idx, a.KV, a.recip_KV);
      r.g = idx - e * a.KV;
      r.x = a.items[2 * e];
      r.y = a.items[2 * e + 1];
    }
    return r;
  };

  if (warp < 4) {
    warpgroup_reg_dealloc<REG_CTRL>();
    if (warp == 0) {
      // ---------------- K / V tiles ----------------
      if (lane == 0) {
        prefetch_tensormap(&tmQ);
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
        int kt = 0;
        bool ok = true;
        RawItem next = load_item(0);
        for (int k = 0; ok && next.g >= 0; k++) {
          const Item it = unpack(next);
          next = load_item(k + 1);
          for (int j = 0; j < it.ntiles; j++, kt++) {
            const int s = kt % KV_STAGES;
            const uint32_t before = ((kt - KV_STAGES) / KV_STAGES) & 1;
            uint8_t* st = kvsm + s * KV_STAGE;
            const int row = it.k0 + it.n_first + j * BN;
            if (kt >= KV_STAGES && !mbar_wait(&bars[kKEmpty + s], before, a.status)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&bars[kKFull + s], TILE);
            tma_load_3d(st, &tmK, &bars[kKFull + s], 0, it.g, row);
            tma_load_3d(st + BOX, &tmK, &bars[kKFull + s], 64, it.g, row);
            if (kt >= KV_STAGES && !mbar_wait(&bars[kVEmpty + s], before, a.status)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&bars[kVFull + s], TILE);
            tma_load_3d(st + TILE, &tmV, &bars[kVFull + s], 0, it.g, row);
            tma_load_3d(st + TILE + BOX, &tmV, &bars[kVFull + s], 64, it.g, row);
          }
        }
      }
    } else if (warp == 3) {
      // ---------------- query tiles: one TMA box, or where 128 rows are no whole queries, row by row ----------------
      // (rows behind the sequence's last are anything: they stay within themselves and are not stored)
      int qn = 0;
      bool ok = true;
      RawItem next = load_item(0);
      for (int k = 0; ok && next.g >= 0; k++) {
        const Item it = unpack(next);
        next = load_item(k + 1);
        for (int hd = 0; hd < 2; hd++, qn++) {
          const int slot = qn % Q_SLOTS;
          if (qn >= Q_SLOTS && !wait(kQEmpty + slot, ((qn - Q_SLOTS) / Q_SLOTS) & 1)) {
            ok = false;
            break;
          }
          if (a.q_tma) {
            if (lane == 0) {
              uint8_t* box = qsm + slot * TILE;
              const int q = it.q0 + quot(it.r0 + hd * BM, a.G, a.recip_G);
              mbar_arrive_expect_tx(&bars[kQFull + slot], TILE);
              tma_load_3d(box, &tmQ, &bars[kQFull + slot], 0, it.g * a.G, q);
              tma_load_3d(box + BOX, &tmQ, &bars[kQFull + slot], 64, it.g * a.G, q);
            }
            continue;
          }
          const uint32_t dst = smem_u32(qsm + slot * TILE);
          const int piece = lane & 15;  // 16 bytes of a row
          int q = quot(it.r0 + hd * BM + (lane >> 4), a.G, a.recip_G), h = it.r0 + hd * BM + (lane >> 4) - q * a.G;  // row's query and head
#pragma unroll 4
          for (int i = 0; i < 64; i++) {
            const int row = (lane >> 4) + 2 * i;
            const bool there = q < it.lq;
            const T* src = static_cast<const T*>(a.q) + (long long)(it.q0 + (there ? q : 0)) * a.q_stride + (long long)(it.g * a.G + h) * HD + piece * 8;
            copy16(dst + (piece >> 3) * BOX + sw128_offset(row, (piece & 7) * 16), src, there);
            for (h += 2; h >= a.G; h -= a.G) q++;
          }
          copy_commit();
          copy_wait<0>();
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) bar_arrive(bar(kQFull + slot));
        }
      }
    } else {
      // ---------------- MMA issue of a half (warps 1 and 2): the warp walks, one elected lane issues ----------------
      const int hd = warp - 1;
      const bool leader = elect_one_sync();
      auto wait = [&](int i, uint32_t parity) { return bar_wait<true>(bar0 + 8 * i, parity, a.status); };
      constexpr uint32_t idesc_qk = idesc_f16(BM, BN, BF16, false, false);
      constexpr uint32_t idesc_pv = idesc_f16(BM, HD, BF16, false, true);
      // Descriptors: the first k-step's, to which a constant per k-step is added.
      const uint64_t dq = smem_desc_sw128(smem_u32(qsm), 16, 1024), dk = smem_desc_sw128(smem_u32(kvsm), 16, 1024);
      const uint64_t dv = smem_desc_sw128(smem_u32(kvsm) + TILE, BOX, 1024);  // MN-major
      const uint32_t ts = tmem + kColS, tp = tmem + kColP + hd * 64, to = tmem + hd * HD;
      // Value rows behind the sequence's end become zeros (they meet P = 0, but may hold anything).  Both halves' warps
      // write them, each before its own products: the same zeros.
      auto clean = [&](int valid, int s) {
        uint8_t* v = kvsm + s * KV_STAGE + TILE;
        for (int i = valid * 8 + lane; i < BN * 8; i += 32) {
          *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(v + BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async();
        __syncwarp();
      };
      // S = Q K^T runs one tile ahead of O += P V.  The scores' place: tile st, tile sj of sn in its item, whose query
      // tile is number sq.
      int st = 0, sj = 0, sn = 0, sq = hd;
      RawItem next = load_item(0);
      int valid = BN;  // keys of the last tile of the item that the scores are in
      auto enter = [&]() {
        const Item it = unpack(next);
        sn = it.ntiles, sj = 0;
        valid = max(0, it.lk - it.n_first - (it.ntiles - 1) * BN);
      };
      bool ok = true, more = next.g >= 0;
      if (more) {
        enter();
        next = load_item(1);
      }
      int k = 1;  // item that `next` holds
      auto scores = [&]() -> bool {
        const int s = st % KV_STAGES, slot = sq % Q_SLOTS;
        if (!wait(kKFull + s, (st / KV_STAGES) & 1) || (sj == 0 && !wait(kQFull + slot, (sq / Q_SLOTS) & 1)) ||
            (st + hd > 0 && !wait(kSRead + (hd ^ 1), (st + hd - 1) & 1)))
          return false;
        tc_fence_after();
        const uint64_t ad = dq + slot * (TILE >> 4), bd = dk + s * (KV_STAGE >> 4);
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
          const uint64_t x = ad + (((ks >> 2) * BOX + (ks & 3) * 32) >> 4), y = bd + (((ks >> 2) * BOX + (ks & 3) * 32) >> 4);
          if (leader) mma_f16_ss(ts, x, y, idesc_qk, ks > 0);
        }
        if (leader) {
          bar_commit(bar(kSFull + hd));
          bar_commit(bar(kKEmpty + s));
          if (sj + 1 == sn) bar_commit(bar(kQEmpty + slot));
        }
        st++;
        if (++sj == sn) {
          sq += 2;
          more = next.g >= 0;
          if (more) {
            enter();
            next = load_item(++k);
          }
        }
        return true;
      };
      int pj = 0, pn = sn, pvalid = valid, items = 0;  // the products' place: tile pj of pn in the items-th item
      if (more) ok = scores();
      for (int t = 0; ok && t < st; t++) {  // tile t: its scores have been issued
        const int sn1 = sn, valid1 = valid;  // of the item of the tile after this one
        if (more && !scores()) break;
        const int s = t % KV_STAGES;
        if (!wait(kVFull + s, (t / KV_STAGES) & 1)) break;
        if (pj + 1 == pn && pvalid < BN) clean(pvalid, s);
        // O += P V in two halves of 64 keys: the first runs while the softmax computes the second half of P
        const uint64_t vd = dv + s * (KV_STAGE >> 4);
        if (!wait(kPHalf + hd, t & 1) || (pj == 0 && items > 0 && !wait(kOFree + hd, (items - 1) & 1))) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
          const uint64_t y = vd + ks * (2048 >> 4);
          if (leader) mma_f16_ts(to, tp + ks * 8, y, idesc_pv, (pj > 0 || ks > 0) ? 1u : 0u);
        }
        if (!wait(kPFull + hd, t & 1)) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 4; ks < 8; ks++) {
          const uint64_t y = vd + ks * (2048 >> 4);
          if (leader) mma_f16_ts(to, tp + ks * 8, y, idesc_pv, 1u);
        }
        if (leader) {
          bar_commit(bar(kPVDone + hd));
          bar_commit(bar(kVEmpty + s));
        }
        if (++pj == pn) {
          pj = 0, pn = sn1, pvalid = valid1, items++;
        }
      }
    }
  } else {
    // ---------------- softmax of one half, one thread per row ----------------
    warpgroup_reg_alloc<REG_SOFTMAX>();
    const int hd = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t sc = tmem + lane_off + kColS, pc = tmem + lane_off + kColP + hd * 64, oc = tmem + lane_off + hd * HD;
    // A finished item's result: out of TMEM and into the output.  It runs after the NEXT item's first P is in TMEM, which
    // waited for the finished item's last product.
    int f_row = -1, f_head = 0;  // this thread's finished row: query row (-1: none), head
    bool f_empty = false;        // it sees no key
    float f_l = 0.f;
    bool fin = false;
    auto epilogue = [&]() {
      const bool sum = f_l > 0.f && f_l < INFINITY;  // else the row is NaN, whatever its values are
      const float inv = 1.f / f_l;
      const uint64_t inv2 = f2(inv, inv);
      uint32_t top = 0u;  // largest magnitude of the stored elements, by their bits
      T* dst = static_cast<T*>(a.out) + ((long long)f_row * a.H + f_head) * HD;
#pragma unroll 1
      for (int c = 0; c < 4; c++) {
        uint32_t o[32];
        tmem_ld32(oc + 32 * c, o);
        tmem_ld_wait();
        float w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float y0, y1;
          f2_get(f2_mul(f2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), inv2), y0, y1);
          const uint32_t y = pack16<BF16>(y0, y1);
          top = __vmaxu2(top, y & 0x7fff7fffu);
          w[i] = __uint_as_float(f_empty ? 0u : sum ? y : kNoSum);
        }
        if (f_row >= 0) {
          st_global_v8(reinterpret_cast<float*>(dst + 32 * c), w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
          st_global_v8(reinterpret_cast<float*>(dst + 32 * c + 16), w[8], w[9], w[10], w[11], w[12], w[13], w[14], w[15]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(bar(kOFree + hd));
      const bool bad = f_row >= 0 && !f_empty && sum && not_finite<BF16>(top);
      if (__any_sync(0xffffffffu, bad) && lane == 0) s_mend[hd].any = 1;
      fin = false;
    };
    int nt = 0;  // key tiles of this half so far
    bool ok = true;
    RawItem next = load_item(0);
    for (int k = 0; ok && next.g >= 0; k++) {
      const Item it = unpack(next);
      next = load_item(k + 1);
      const int first = it.r0 + hd * BM, r = first + row, qi = quot(r, a.G, a.recip_G), pos = it.lk - it.lq + qi;
      const int q_first = quot(first, a.G, a.recip_G), q_last = min(it.lq - 1, quot(first + BM - 1, a.G, a.recip_G));
      const bool exists = qi < it.lq;
      // every row of the half sees keys [all_lo, all_hi]
      const int all_hi = q_first < it.lq ? it.lk - it.lq + q_first : -1;
      const int all_lo = a.window > 0 ? it.lk - it.lq + q_last - a.window + 1 : 0;
      const int row_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0, row_hi = exists ? pos : -1;
      float m_use = -INFINITY, l = 0.f;
      for (int j = 0; j < it.ntiles; j++) {
        const int t = nt + j, n0 = it.n_first + j * BN;
        if (!wait(kSFull + hd, t & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const bool full = n0 >= all_lo && n0 + BN - 1 <= all_hi;
        const int lo = row_lo - n0, hi = row_hi - n0;
        uint32_t s0[32], s1[32], s2[32], s3[32];
        tmem_ld32(sc, s0);
        tmem_ld32(sc + 32, s1);
        tmem_ld32(sc + 64, s2);
        tmem_ld32(sc + 96, s3);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(kSRead + hd));
        bool e0 = false, e1 = false, e2 = false, e3 = false;
        if (!full) {
          e0 = mask_chunk<0>(s0, lo, hi);
          e1 = mask_chunk<32>(s1, lo, hi);
          e2 = mask_chunk<64>(s2, lo, hi);
          e3 = mask_chunk<96>(s3, lo, hi);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (!e0) chunk_max(s0, mx4);
        if (!e1) chunk_max(s1, mx4);
        if (!e2) chunk_max(s2, mx4);
        if (!e3) chunk_max(s3, mx4);
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
        const bool move = mx > m_use + RESCALE_LOG2 || (j == 0 && mx > m_use);
        const bool rescale_o = move && j > 0 && m_use != -INFINITY;
        const float f = rescale_o ? ex2_approx(m_use - mx) : 1.f;
        // P and O are this thread's again once the product of the tile before is done: asked for here, needed when P is there.
        const bool pv_done = t == 0 || bar_try(bar(kPVDone + hd), (t - 1) & 1);
        if (__any_sync(0xffffffffu, rescale_o)) {
          if (t > 0 && !wait(kPVDone + hd, (t - 1) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 4; c++) {
            uint32_t r32[32];
            tmem_ld32(oc + 32 * c, r32);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i++) r32[i] = __float_as_uint(__uint_as_float(r32[i]) * f);
            tmem_st32(oc + 32 * c, r32);
          }
          tmem_st_wait();
        }
        if (move) {
          l *= f;
          m_use = mx;
        }
        const float neg_m = m_use == -INFINITY ? 0.f : -m_use;
        const uint64_t scale2 = f2(a.scale_log2, a.scale_log2), negm2 = f2(neg_m, neg_m);
        uint64_t ls2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
        auto half_p = [&](const uint32_t (&x)[32], bool ex, const uint32_t (&y)[32], bool ey, uint32_t col, int done) {
          uint32_t pk[32];
          chunk_p<BF16, 0>(x, ex, scale2, negm2, ls2, pk);
          chunk_p<BF16, 16>(y, ey, scale2, negm2, ls2, pk);
          if (col == 0) {
            if (!__all_sync(0xffffffffu, pv_done) && !wait(kPVDone + hd, (t - 1) & 1)) ok = false;
            tc_fence_after();
          }
          tmem_st32(pc + col, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(bar(done));
        };
        half_p(s0, e0, s1, e1, 0, kPHalf + hd);
        half_p(s2, e2, s3, e3, 32, kPFull + hd);
        float a0, a1, b0, b1;
        f2_get(ls2[0], a0, a1);
        f2_get(ls2[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
        if (!ok) break;
        if (j == 0 && fin) epilogue();
      }
      if (!ok) break;
      fin = true;
      f_row = exists ? it.q0 + qi : -1;
      f_head = it.g * a.G + r - qi * a.G;
      f_empty = row_lo > row_hi;
      f_l = l;
      nt += it.ntiles;
    }
    if (ok && fin && wait(kPVDone + hd, (nt - 1) & 1)) {
      tc_fence_after();
      epilogue();
    }
    if (!ok && lane == 0) s_mend[hd].late = 1;
    half_sync(hd);  // the half's results are stored
    if (s_mend[hd].any && !s_mend[hd].late) {
      RawItem next = load_item(0);
      for (int k = 0; next.g >= 0; k++) {
        const Item it = unpack(next);
        next = load_item(k + 1);
        mend_rows<BF16>(a, it, hd, row, s_mend[hd]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

constexpr size_t kSmem = 1024 + Q_SLOTS * TILE + KV_STAGES * KV_STAGE;
static_assert(kSmem <= 227 * 1024, "shared memory");

template <bool BF16>
int launch(hcu_context* h, const VarlenArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, int grid) {
  const char* op = "hcu_prefill_varlen";
  auto kern = prefill_varlen_kernel<BF16>;
  static std::atomic<uint64_t> attr_done{0};  // per device
  HCU_TRY(once_per_device(attr_done, h->device, [&]() -> int {
    return check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem), op);
  }));
  if (!a.direct) {
    varlen_items_kernel<<<1, 1024, 0, h->stream>>>(a);
    HCU_TRY(after_launch("hcu_prefill_varlen: items"));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = h->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set up while the items are sorted
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.direct ? 0 : 1;
  (void)cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, a);
  return after_launch("hcu_prefill_varlen: launch");  // takes the error, so that no later call finds it
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
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 ||
      reinterpret_cast<uintptr_t>(out) % 32)
    return fail(HCU_EINVAL, "%s: q, k and v must be 16-byte, out 32-byte aligned", op);
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
  // A window as long as the longest sequence hides nothing (and the first key's index minus a larger one could pass 2^31).
  a.window = p->window >= p->total_k ? 0 : (int)p->window;
  a.recip_G = (uint32_t)std::min<uint64_t>(0xffffffffull, (1ull << 32) / a.G + 1);
  a.recip_KV = (uint32_t)std::min<uint64_t>(0xffffffffull, (1ull << 32) / a.KV + 1);
  a.total_q = (int)p->total_q;
  a.total_k = (int)p->total_k;
  a.scale_log2 = hcu::kLog2e / sqrtf(128.f);
  a.status = h->dev_status;
  // The item list lives in the workspace, behind the other ops' tickets.
  const long long most = ((long long)a.total_q * a.G + 2 * hcu::BM - 1) / (2 * hcu::BM) + a.batch;  // blocks of 256 rows
  const size_t offsets = ((size_t)(a.batch + 1) * sizeof(int) + 15) / 16 * 16, need = hcu::kTicketBytes + offsets + (size_t)most * 2 * sizeof(int4);
  if (most * a.KV > 0x3fffffffLL || (long long)a.total_q * a.G > 0x3fffffffLL) return fail(HCU_EINVAL, "%s: too many rows", op);
  if (need > h->workspace_bytes)
    return fail(HCU_ENOMEM, "%s: the list of %lld blocks needs a workspace of %zu bytes (this one has %zu)", op, most, need, h->workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(h->workspace) + hcu::kTicketBytes;
  a.blocks = reinterpret_cast<int*>(ws);
  a.items = reinterpret_cast<int4*>(ws + offsets);
  // Without any key the K and V maps cover a row of q (all of whose "keys" are masked).
  CUtensorMap tq, tk, tv;
  const CUtensorMapDataType dt = p->dtype == HCU_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto map = [&](CUtensorMap* m, const void* base, int heads, long long rows, long long stride, uint32_t box_heads, uint32_t box_rows) {
    const uint64_t dims[3] = {128, (uint64_t)heads, (uint64_t)rows};
    const uint64_t strides[2] = {256, (uint64_t)stride * 2};
    const uint32_t box[3] = {64, box_heads, box_rows};
    return hcu::make_tensor_map(m, dt, 3, const_cast<void*>(base), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  HCU_TRY(map(&tk, a.total_k ? k : q, a.KV, a.total_k ? a.total_k : 1, a.k_stride, 1, 128));
  HCU_TRY(map(&tv, a.total_k ? v : q, a.KV, a.total_k ? a.total_k : 1, a.v_stride, 1, 128));
  a.q_tma = a.G <= 128 && 128 % a.G == 0;
  HCU_TRY(map(&tq, q, a.H, a.total_q, a.q_stride, a.q_tma ? (uint32_t)a.G : 1, a.q_tma ? 128u / a.G : 1));
  int grid = (int)std::min<long long>(h->sm_count, most * a.KV);
  if (h->opt_swa_ctas > 0 && h->opt_swa_ctas < grid) grid = (int)h->opt_swa_ctas;
  a.direct = most * a.KV <= grid && a.batch <= hcu::kDirectBatch;
  return p->dtype == HCU_DT_BF16 ? hcu::launch<true>(h, a, tq, tk, tv, grid) : hcu::launch<false>(h, a, tq, tk, tv, grid);
}
