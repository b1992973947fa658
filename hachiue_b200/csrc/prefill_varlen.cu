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
//    whatever the lengths are.
//  * Warp roles: K / V by TMA (warp 0), tcgen05.mma (warp 1), Q rows by cp.async
//    (warps 2, 3), and a softmax warpgroup per tile, one thread per row.  S is in
//    TMEM, P goes back over its columns, O stays in TMEM across the keys.  While
//    one tile's softmax runs the tensor cores work on the other tile.
//  * Half of the exponentials of a tile without a mask run on the FMA pipe: 2^x =
//    2^n 2^f with n = round(x) and a cubic minimax polynomial for 2^f (relative
//    error 7.5e-5, below the 2^-12 of rounding P to f16), so that the SFU takes half the time.
//  * O is rescaled only when a row's maximum grows by more than 2^8: P stays
//    below 2^8 otherwise and O / l cancels the stale maximum.
//  * Keys and values behind a sequence's end have no influence: scores are
//    selected, value rows are zeroed in shared memory.  Masked keys inside the sequence
//    meet P = 0; where such a value is not finite the row's result is not either, and
//    the row is computed again over its visible keys alone (slow, exact, never taken by finite inputs).
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
  int4* items;       // [2 * blocks]: {first query, queries, first key, keys}, {block of the sequence, 0, 0, 0}
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
// and writes them out.  Sequences whose offsets are not in order or not within the tensors are reported and left out.
__global__ void __launch_bounds__(1024) varlen_items_kernel(const VarlenArgs a) {
  __shared__ int bins[kBins], part[32], base;
  asm volatile("griddepcontrol.launch_dependents;");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  bins[tid] = 0;
  if (tid == 0) base = 0;
  __syncthreads();
  for (int b0 = 0; b0 < a.batch; b0 += 1024) {
    const int b = b0 + tid;
    int n = 0;
    if (b < a.batch) {
      const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
      if (q0 < 0 || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) atomicOr(a.status, HCU_DEVERR_BADARG);
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
    if (tid == 1023) base = before + pre;
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
      const int r1 = (int)min((long long)lq * a.G, (blk + 1) * 2LL * BM);
      const int cost = key_tiles(blk * 2 * BM, r1, a.G, lq, lk, a.window).y;
      const int bin = kBins - 1 - min(cost, kBins - 1);
      if (pass == 0) {
        atomicAdd(&bins[bin], 1);
      } else {
        const int at = atomicAdd(&bins[bin], 1);
        a.items[2 * at] = make_int4(q0, lq, k0, lk);
        a.items[2 * at + 1] = make_int4(blk, 0, 0, 0);
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
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 2^x for two x <= 127 on the FMA pipe: n = round(x) by adding 1.5 * 2^23, f = x - n in [-1/2, 1/2], a cubic for 2^f
// (minimax fit of the relative error), and n added to the exponent.  Below -126 the result is near 2^-126; NaN gives
// something not finite once rounded to 16 bits.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float x0, x1;
  f2_get(x, x0, x1);
  x = f2(fmax_nan(x0, -126.f), fmax_nan(x1, -126.f));
  const uint64_t magic = f2(12582912.f, 12582912.f), unmagic = f2(-12582912.f, -12582912.f);
  const uint64_t t = f2_add(x, magic);
  const uint64_t f = f2_fma(f2_add(t, unmagic), f2(-1.f, -1.f), x);
  uint64_t p = f2_fma(f2(0.0551716649f, 0.0551716649f), f, f2(0.242611122f, 0.242611122f));
  p = f2_fma(p, f, f2(0.693260986f, 0.693260986f));
  p = f2_fma(p, f, f2(0.999928074f, 0.999928074f));
  float t0, t1, p0, p1;
  f2_get(t, t0, t1);
  f2_get(p, p0, p1);
  return f2(__uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23)),
            __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23)));
}

// Scores of columns outside lo..hi (tile columns) become -inf, in one 32-column chunk beginning at column C0.  Returns
// whether no row of the warp keeps any column of it (warp-uniform; the chunk is then left as it is and skipped).
template <int C0>
__device__ __forceinline__ bool mask_chunk(uint32_t (&r)[32], int lo, int hi) {
  if (__all_sync(0xffffffffu, lo <= C0 && hi >= C0 + 31)) return false;
  if (__all_sync(0xffffffffu, hi < C0 || lo > C0 + 31)) return true;
  const int a = lo - C0, b = hi - C0;
#pragma unroll
  for (int i = 0; i < 32; i++) r[i] = (i >= a && i <= b) ? r[i] : 0xff800000u;  // -inf
  return false;
}
__device__ __forceinline__ void chunk_max(const uint32_t (&r)[32], float (&mx)[4]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2)
    mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
}

#ifndef POLY
#define POLY 2
#endif
// P of one 32-column chunk as 16 words pk[OFF..], added to the row's sums.  With FULL (no mask in the tile) every second
// pair takes the FMA pipe's exponential.
template <bool BF16, bool FULL, int OFF>
__device__ __forceinline__ void chunk_p(const uint32_t (&r)[32], bool empty, uint64_t scale2, uint64_t negm2, uint64_t (&ls2)[2],
                                        uint32_t (&pk)[32]) {
  if (empty) {
#pragma unroll
    for (int i = 0; i < 16; i++) pk[OFF + i] = 0u;
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; i++) {
    uint64_t x = f2_fma(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), scale2, negm2);
    float p0, p1;
    if (FULL && POLY > 0 && i % POLY == POLY - 1) {
      x = exp2_pair(x);
      f2_get(x, p0, p1);
    } else {
      float v0, v1;
      f2_get(x, v0, v1);
      p0 = ex2_approx(v0), p1 = ex2_approx(v1);
      x = f2(p0, p1);
    }
    ls2[i & 1] = f2_add(ls2[i & 1], x);
    pk[OFF + i] = pack16<BF16>(p0, p1);
  }
}

// One row over its visible keys [lo, hi], by a warp: for rows that a value outside them made not finite.
template <typename T>
__device__ __noinline__ void row_alone(const VarlenArgs& a, int q_row, int head, int k0, int lo, int hi) {
  const int lane = threadIdx.x & 31, g = head / a.G;
  float q[4], acc[4] = {}, m = -INFINITY, l = 0.f;
  load4(static_cast<const T*>(a.q) + (long long)q_row * a.q_stride + head * HD + 4 * lane, q);
  for (int t = lo; t <= hi; t++) {
    float k[4], v[4];
    load4(static_cast<const T*>(a.k) + (long long)(k0 + t) * a.k_stride + g * HD + 4 * lane, k);
    load4(static_cast<const T*>(a.v) + (long long)(k0 + t) * a.v_stride + g * HD + 4 * lane, v);
    float x = fmaf(q[0], k[0], fmaf(q[1], k[1], fmaf(q[2], k[2], q[3] * k[3])));
    x = warp_sum(x) * a.scale_log2;
    const float mn = fmaxf(m, x), f = exp2f(m - mn), p = exp2f(x - mn);
    m = mn;
    l = fmaf(l, f, p);
#pragma unroll
    for (int c = 0; c < 4; c++) acc[c] = fmaf(acc[c], f, p * v[c]);
  }
#pragma unroll
  for (int c = 0; c < 4; c++) acc[c] /= l;
  store4(static_cast<T*>(a.out) + ((long long)q_row * a.H + head) * HD + 4 * lane, acc);
}

// A work item: 256 packed rows of one sequence and KV head.
struct Item {
  int q0, lq, k0, lk, g, r0;  // first query and their number, first key and their number, KV head, first packed row
  int n_first, ntiles;        // first key of the first tile, tiles of the item
  int nt[2];                  // tiles of each half (0: the half has no row)
};

__device__ __forceinline__ Item get_item(const VarlenArgs& a, int idx) {
  const int e = idx / a.KV;
  const int4 x = a.items[2 * e];
  Item it;
  it.q0 = x.x, it.lq = x.y, it.k0 = x.z, it.lk = x.w;
  it.g = idx % a.KV;
  it.r0 = a.items[2 * e + 1].x * 2 * BM;
  const int rows = (int)min((long long)it.lq * a.G - it.r0, 2LL * BM);
  const int2 both = key_tiles(it.r0, it.r0 + rows, a.G, it.lq, it.lk, a.window);
  it.n_first = both.x, it.ntiles = both.y;
  const int last0 = it.lk - it.lq + (it.r0 + min(rows, BM) - 1) / a.G;  // position of the first half's last row
  it.nt[0] = rows > BM ? (last0 < it.n_first ? 1 : (last0 - it.n_first) / BN + 1) : it.ntiles;
  it.nt[1] = rows > BM ? it.ntiles : 0;
  return it;
}

// The k-th item of this CTA: rounds of gridDim.x items, forwards in even rounds and backwards in odd ones (costs fall
// with the index).
__device__ __forceinline__ int item_index(int k) {
  const int P = (int)gridDim.x, c = (int)blockIdx.x;
  return k * P + ((k & 1) ? P - 1 - c : c);
}

// Barriers run on across items; every role advances the same counters:
//   q_full / q_empty   per query tile (slot = tiles so far mod 3),
//   kv_full / kv_empty per key tile of the items (ring),
//   s_full, p_half, p_full per key tile and half,
//   o_free             per item and half: O has been read, the next P.V may overwrite it,
//   o_done             at the end.
template <bool BF16>
__global__ void __launch_bounds__(384, 1)
    prefill_varlen_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const VarlenArgs a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qsm = smem;                    // [Q_SLOTS][TILE]
  uint8_t* kvsm = qsm + Q_SLOTS * TILE;   // [KV_STAGES][K tile | V tile]
  __shared__ uint64_t q_full[Q_SLOTS], q_empty[Q_SLOTS], kv_full[KV_STAGES], kv_empty[KV_STAGES];
  __shared__ uint64_t s_full[2], p_half[2], p_full[2], o_free[2], o_done;
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < Q_SLOTS; i++) mbar_init(&q_full[i], 2), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < KV_STAGES; i++) mbar_init(&kv_full[i], 1), mbar_init(&kv_empty[i], 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_half[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_free[i], 4);
    }
    mbar_init(&o_done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // TMEM columns per half: S (P over its first 64 columns), then O.
  auto s_col = [](int hd) { return (uint32_t)(hd * 256); };
  auto o_col = [](int hd) { return (uint32_t)(hd * 256 + 128); };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_items = a.blocks[a.batch] * a.KV;

  if (warp < 4) {
    warpgroup_reg_dealloc<REG_CTRL>();
    if (warp == 0) {
      // ---------------- K / V tiles ----------------
      if (lane == 0) {
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
        int kt = 0;
        bool ok = true;
        for (int k = 0; ok; k++) {
          const int idx = item_index(k);
          if (idx >= n_items) break;
          const Item it = get_item(a, idx);
          for (int j = 0; j < it.ntiles; j++, kt++) {
            const int s = kt % KV_STAGES;
            if (kt >= KV_STAGES && !mbar_wait(&kv_empty[s], ((kt - KV_STAGES) / KV_STAGES) & 1, a.status)) {
              ok = false;
              break;
            }
            uint8_t* st = kvsm + s * KV_STAGE;
            const int row = it.k0 + it.n_first + j * BN;
            mbar_arrive_expect_tx(&kv_full[s], KV_STAGE);
            tma_load_3d(st, &tmK, &kv_full[s], 0, it.g, row);
            tma_load_3d(st + BOX, &tmK, &kv_full[s], 64, it.g, row);
            tma_load_3d(st + TILE, &tmV, &kv_full[s], 0, it.g, row);
            tma_load_3d(st + TILE + BOX, &tmV, &kv_full[s], 64, it.g, row);
          }
        }
      }
    } else if (warp >= 2) {
      // ---------------- query tiles: rows of any stride, zeros behind the last ----------------
      int qn = 0;
      bool ok = true;
      for (int k = 0; ok; k++) {
        const int idx = item_index(k);
        if (idx >= n_items) break;
        const Item it = get_item(a, idx);
        for (int hd = 0; hd < 2 && it.nt[hd] > 0; hd++, qn++) {
          const int slot = qn % Q_SLOTS;
          if (qn >= Q_SLOTS && !__all_sync(0xffffffffu, mbar_wait(&q_empty[slot], ((qn - Q_SLOTS) / Q_SLOTS) & 1, a.status))) {
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(qsm + slot * TILE);
          const int piece = lane & 15;  // 16 bytes of a row
#pragma unroll 4
          for (int i = 0; i < 32; i++) {
            const int row = (warp - 2) * 2 + (lane >> 4) + 4 * i, r = it.r0 + hd * BM + row;
            const int q = r / a.G, h = it.g * a.G + r % a.G;
            const bool there = q < it.lq;
            const T* src = static_cast<const T*>(a.q) + (long long)(it.q0 + (there ? q : 0)) * a.q_stride + (long long)h * HD + piece * 8;
            copy16(dst + (piece >> 3) * BOX + sw128_offset(row, (piece & 7) * 16), src, there);
          }
          copy_commit();
          copy_wait<0>();
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[slot]);
        }
      }
    } else {
      // ---------------- MMA issue: the warp walks, one elected lane issues ----------------
      const bool leader = elect_one_sync();
      constexpr uint32_t idesc_qk = idesc_f16(BM, BN, BF16, false, false);
      constexpr uint32_t idesc_pv = idesc_f16(BM, HD, BF16, false, true);
      const uint32_t qb = smem_u32(qsm), kvb = smem_u32(kvsm);
      auto qk = [&](int hd, int slot, int s) {
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
          const uint64_t ad = smem_desc_sw128(qb + slot * TILE + (ks >> 2) * BOX + (ks & 3) * 32, 16, 1024);
          const uint64_t bd = smem_desc_sw128(kvb + s * KV_STAGE + (ks >> 2) * BOX + (ks & 3) * 32, 16, 1024);
          if (leader) mma_f16_ss(tmem + s_col(hd), ad, bd, idesc_qk, ks > 0);
        }
        if (leader) mma_commit(&s_full[hd]);
      };
      auto pv_half = [&](int hd, int s, int half, bool acc) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int ks = 4 * half + i;
          const uint64_t bd = smem_desc_sw128(kvb + s * KV_STAGE + TILE + ks * 2048, BOX, 1024);  // MN-major V
          if (leader) mma_f16_ts(tmem + o_col(hd), tmem + s_col(hd) + ks * 8, bd, idesc_pv, (acc || ks > 0) ? 1u : 0u);
        }
      };
      // Value rows behind the sequence's end become zeros (they meet P = 0, but may hold anything).
      auto clean = [&](const Item& it, int j, int s) {
        const int valid = max(0, it.lk - it.n_first - j * BN);
        if (valid >= BN) return;
        uint8_t* v = kvsm + s * KV_STAGE + TILE;
        for (int i = valid * 8 + lane; i < BN * 8; i += 32) {
          *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(v + BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async();
        __syncwarp();
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_poll(bar, parity, a.status)); };
      int kt = 0, qn = 0;        // key tiles and query tiles so far, this item's first
      int nt[2] = {0, 0};        // key tiles of each half so far
      int done[2] = {0, 0};      // items of each half so far
      bool ok = true;
      int idx = item_index(0);
      Item it{};
      if (idx < n_items) {
        it = get_item(a, idx);
        ok = wait(&kv_full[0], 0);
        for (int hd = 0; ok && hd < 2 && it.nt[hd] > 0; hd++) {
          ok = wait(&q_full[hd], 0);
          if (!ok) break;
          tc_fence_after();
          qk(hd, hd, 0);
          if (it.nt[hd] == 1 && leader) mma_commit(&q_empty[hd]);
          if (hd == 0) clean(it, 0, 0);
        }
      }
      for (int k = 0; ok && idx < n_items; k++) {
        idx = item_index(k + 1);
        const bool more = idx < n_items;
        const Item next = more ? get_item(a, idx) : it;
        const int qn1 = qn + (it.nt[1] > 0 ? 2 : 1);
        for (int j = 0; ok && j < it.ntiles; j++) {
          const int s = (kt + j) % KV_STAGES, s1 = (kt + j + 1) % KV_STAGES, last_half = it.nt[1] > 0 ? 1 : 0;
          const bool last = j + 1 == it.ntiles;
          bool cleaned = false;
          for (int hd = 0; hd < 2; hd++) {
            if (j < it.nt[hd]) {
              const int t = nt[hd] + j;
              if (!wait(&p_half[hd], t & 1) || (j == 0 && done[hd] > 0 && !wait(&o_free[hd], (done[hd] - 1) & 1))) {
                ok = false;
                break;
              }
              tc_fence_after();
              pv_half(hd, s, 0, j > 0);
              if (!wait(&p_full[hd], t & 1)) {
                ok = false;
                break;
              }
              tc_fence_after();
              pv_half(hd, s, 1, true);
              if (hd == last_half && leader) mma_commit(&kv_empty[s]);
            }
            // The half's next scores overwrite its P: behind the P.V above.  At the item's last tile: the next item's first.
            const bool here = j + 1 < it.nt[hd], there = last && more && next.nt[hd] > 0;
            if (here || there) {
              const int q = here ? qn + hd : qn1 + hd;
              if (!wait(&kv_full[s1], ((kt + j + 1) / KV_STAGES) & 1) || (there && !wait(&q_full[q % Q_SLOTS], (q / Q_SLOTS) & 1))) {
                ok = false;
                break;
              }
              tc_fence_after();
              qk(hd, q % Q_SLOTS, s1);
              if ((here ? j + 2 == it.nt[hd] : next.nt[hd] == 1) && leader) mma_commit(&q_empty[q % Q_SLOTS]);
              if (!cleaned) {
                clean(here ? it : next, here ? j + 1 : 0, s1);
                cleaned = true;
              }
            }
          }
        }
        for (int hd = 0; hd < 2; hd++) nt[hd] += it.nt[hd], done[hd] += it.nt[hd] > 0;
        kt += it.ntiles;
        qn = qn1;
        it = next;
      }
      if (leader) mma_commit(&o_done);
    }
  } else {
    // ---------------- softmax of one half, one thread per row ----------------
    warpgroup_reg_alloc<REG_SOFTMAX>();
    const int hd = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t sc = tmem + lane_off + s_col(hd), oc = tmem + lane_off + o_col(hd);
    // A finished item's result: out of TMEM and into the output.  It runs after the NEXT item's first P is in TMEM (O
    // has long been complete by then: the next scores follow the last P.V), so that tile's products cover it.
    int f_row = -1, f_head = 0, f_k0 = 0, f_lo = 0, f_hi = -1;  // this thread's finished row: query row (-1: none), head, visible keys
    float f_l = 0.f;
    bool fin = false;
    auto epilogue = [&]() {
      uint32_t o[4][32];
#pragma unroll
      for (int c = 0; c < 4; c++) tmem_ld32(oc + 32 * c, o[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[hd]);
      const bool empty = f_lo > f_hi;
      const float inv = empty ? 0.f : 1.f / f_l;
      uint64_t sum = f2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 32; i += 2)  // NaN once anything is not finite
          sum = f2_fma(f2(__uint_as_float(o[c][i]), __uint_as_float(o[c][i + 1])), f2(0.f, 0.f), sum);
      float s0, s1;
      f2_get(sum, s0, s1);
      const bool bad = f_row >= 0 && !empty && !(s0 + s1 == 0.f && f_l > 0.f && f_l < INFINITY);
      if (f_row >= 0 && !bad) {
        T* dst = static_cast<T*>(a.out) + ((long long)f_row * a.H + f_head) * HD;
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            uint32_t* p = &w.x;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float y0 = empty ? 0.f : __uint_as_float(o[c][i + 2 * e]) * inv;
              const float y1 = empty ? 0.f : __uint_as_float(o[c][i + 2 * e + 1]) * inv;
              p[e] = pack16<BF16>(y0, y1);
            }
            *reinterpret_cast<uint4*>(dst + 32 * c + i) = w;
          }
      }
      for (uint32_t rows = __ballot_sync(0xffffffffu, bad); rows; rows &= rows - 1) {
        const int src = __ffs(rows) - 1;
        row_alone<T>(a, __shfl_sync(0xffffffffu, f_row, src), __shfl_sync(0xffffffffu, f_head, src),
                     __shfl_sync(0xffffffffu, f_k0, src), __shfl_sync(0xffffffffu, f_lo, src), __shfl_sync(0xffffffffu, f_hi, src));
      }
      fin = false;
    };
    int nt = 0;  // key tiles of this half so far
    bool ok = true;
    for (int k = 0; ok; k++) {
      const int idx = item_index(k);
      if (idx >= n_items) break;
      const Item it = get_item(a, idx);
      if (it.nt[hd] == 0) continue;
      const int first = it.r0 + hd * BM, r = first + row, qi = r / a.G, pos = it.lk - it.lq + qi;
      const bool exists = qi < it.lq;
      // every row of the half sees keys [all_lo, all_hi]
      const int all_hi = it.lk - it.lq + first / a.G;
      const int all_lo = a.window > 0 ? it.lk - it.lq + min(it.lq - 1, (first + BM - 1) / a.G) - a.window + 1 : 0;
      const int row_lo = a.window > 0 ? max(0, pos - a.window + 1) : 0, row_hi = exists ? pos : -1;
      float m_use = -INFINITY, l = 0.f;
      for (int j = 0; j < it.nt[hd]; j++) {
        const int t = nt + j, n0 = it.n_first + j * BN;
        if (!__all_sync(0xffffffffu, mbar_wait(&s_full[hd], t & 1, a.status))) {
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
        const float f = rescale_o ? exp2f(m_use - mx) : 1.f;
        if (__any_sync(0xffffffffu, rescale_o)) {  // P.V of the tile before has landed (s_full of this tile)
#pragma unroll
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
        auto half_p = [&](const uint32_t (&x)[32], bool ex, const uint32_t (&y)[32], bool ey, uint32_t col, uint64_t* bar) {
          uint32_t pk[32];
          if (full) {
            chunk_p<BF16, true, 0>(x, false, scale2, negm2, ls2, pk);
            chunk_p<BF16, true, 16>(y, false, scale2, negm2, ls2, pk);
          } else {
            chunk_p<BF16, false, 0>(x, ex, scale2, negm2, ls2, pk);
            chunk_p<BF16, false, 16>(y, ey, scale2, negm2, ls2, pk);
          }
          tmem_st32(sc + col, pk);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        };
        half_p(s0, e0, s1, e1, 0, &p_half[hd]);
        half_p(s2, e2, s3, e3, 32, &p_full[hd]);
        float a0, a1, b0, b1;
        f2_get(ls2[0], a0, a1);
        f2_get(ls2[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
        if (j == 0 && fin) epilogue();
      }
      if (!ok) break;
      fin = true;
      f_row = exists ? it.q0 + qi : -1;
      f_head = it.g * a.G + r % a.G;
      f_k0 = it.k0;
      f_lo = row_lo, f_hi = row_hi;
      f_l = l;
      nt += it.nt[hd];
    }
    if (ok && fin && __all_sync(0xffffffffu, mbar_wait(&o_done, 0, a.status))) {
      tc_fence_after();
      epilogue();
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
int launch(hcu_context* h, const VarlenArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, int grid) {
  const char* op = "hcu_prefill_varlen";
  auto kern = prefill_varlen_kernel<BF16>;
  static std::atomic<uint64_t> attr_done{0};  // per device
  HCU_TRY(once_per_device(attr_done, h->device, [&]() -> int {
    return check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem), op);
  }));
  varlen_items_kernel<<<1, 1024, 0, h->stream>>>(a);
  HCU_TRY(after_launch("hcu_prefill_varlen: items"));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(384);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = h->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // set up while the items are sorted
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, tk, tv, a), "hcu_prefill_varlen: launch");
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
  // The item list lives in the workspace, behind the other ops' tickets.
  const long long most = ((long long)a.total_q * a.G + 2 * hcu::BM - 1) / (2 * hcu::BM) + a.batch;  // blocks of 256 rows
  const size_t offsets = ((size_t)(a.batch + 1) * sizeof(int) + 15) / 16 * 16, need = hcu::kTicketBytes + offsets + (size_t)most * 2 * sizeof(int4);
  if (most * a.KV > 0x7fffffffLL) return fail(HCU_EINVAL, "%s: too many rows", op);
  if (need > h->workspace_bytes)
    return fail(HCU_ENOMEM, "%s: the list of %lld blocks needs a workspace of %zu bytes (this one has %zu)", op, most, need, h->workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(h->workspace) + hcu::kTicketBytes;
  a.blocks = reinterpret_cast<int*>(ws);
  a.items = reinterpret_cast<int4*>(ws + offsets);
  CUtensorMap tk, tv;
  for (int i = 0; i < 2; i++) {
    // Without any key the map covers a row of q (all of whose "keys" are masked).
    const void* base = a.total_k ? (i ? v : k) : q;
    const long long stride = i ? a.v_stride : a.k_stride;
    const uint64_t dims[3] = {128, (uint64_t)a.KV, (uint64_t)(a.total_k ? a.total_k : 1)};
    const uint64_t strides[2] = {256, (uint64_t)stride * 2};
    const uint32_t box[3] = {64, 1, 128};
    HCU_TRY(hcu::make_tensor_map(i ? &tv : &tk, p->dtype == HCU_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                 3, const_cast<void*>(base), dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B));
  }
  int grid = (int)std::min<long long>(h->sm_count, most * a.KV);
  if (h->opt_swa_ctas > 0 && h->opt_swa_ctas < grid) grid = (int)h->opt_swa_ctas;
  return p->dtype == HCU_DT_BF16 ? hcu::launch<true>(h, a, tk, tv, grid) : hcu::launch<false>(h, a, tk, tv, grid);
}
