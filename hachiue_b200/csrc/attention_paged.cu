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
//  * Softmax: log2 domain, one pass, per warp, p = 2^(x - M) with a whole number M
//    for each row.  The weighted probabilities of a row and block of 32 dimensions
//    are held times a power of two E of their own, so that the largest lies between
//    2^8 and 2^15 whatever the scales of other blocks and of tokens without weight
//    are, and none is off by more than 2^-32 of it beside its rounding (f16's smallest
//    number is 2^-24).  (With one exponent for all blocks, that of the largest scale,
//    values 2^-18 of another block's were off by 1e-4.)  M and the E move only when a
//    number would pass 2^15.
//
// The work is cut by chunks of 32 tokens, not by sequences: see PagedPlan.  A
// warp fetches its chunks into a ring of its own, two ahead, and never waits for
// another warp until they join their sums.
//
// Measured, bf16, 32 query and 8 KV heads of 128, calls in a row: 64 sequences of 271k
// tokens in all 85 us, 312 MB at 3.7 TB/s; one of 131072 47 us.  Issue-bound: 700
// instructions per chunk at 55 % of the slots, of which the masks and shifts of the codes
// are a quarter; 128 registers allow 16 warps per SM.
#include <algorithm>
#include <cfloat>

#include "paged.cuh"

namespace hcu {
namespace {

struct PagedAttnArgs {
  const void* q;
  void* out;
  PagedKV kv;
  const int32_t* table;
  const int32_t* context;
  int batch, S, H, G, R, nrb, window, max_context, table_stride;
  int min_chunks;    // fewest chunks of 32 tokens worth a CTA of their own
  int split;         // kWarpUnits, kLine or kCluster
  int cluster;       // CTAs of a unit (kCluster)
  float scale_log2;  // log2(e) / sqrt(Dh)
  float* part;       // [gridDim.x][2] records of the units at a CTA's two ends: sums [RB][DH], then (M, l) [RB]
  int4* open;        // [gridDim.x] the unit that begins in a CTA and goes on: parts (0: none), sequence, KV head, row block
  uint32_t* status;
  int dtype;
};

constexpr int NW = 8;          // warps of a CTA
// How the units (a sequence's KV head and row block) are handed out: each to a
// warp (no room for partial sums), by equal pieces of the line of all their
// chunks, or each to a cluster of CTAs, which joins its parts through shared
// memory without a second kernel.  The host takes clusters for short contexts
// and few units: up to four chunks per warp, in up to eight CTAs (replayed graphs, f32, 16 / 8
// heads of 128, cluster / line: one sequence of 256 tokens 8.9 / 11.7 us, of 1024
// 10.2 / 11.7, 16 of 1024 14.7 / 17.1, 16 of 2048 20.3 / 22.6; one of 2048 11.9 / 11.9, of
// 4096 13.8 / 12.3).
constexpr int kWarpUnits = 0, kLine = 1, kCluster = 2;
constexpr int CHUNK = 32;      // tokens a warp takes at a time
constexpr int kUnitCost = 3;    // chunks that a unit's queries and sums cost a warp besides its chunks
constexpr float kNoM = -FLT_MAX;  // M of a row that has seen no token: below every finite score
constexpr int kTop = 15, kStart = 8;  // weighted probabilities stay below 2^kTop; a moved E leaves the largest near 2^kStart
constexpr uint32_t kMostE = 253;      // exponent bits of the largest E, 2^126: that of a block without a weight

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with a zero accumulator.
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Transposes an 8 x 8 matrix of 16-bit elements held one row per four lanes.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// 2^n for n up to 127; 0 below 2^-126.
__device__ __forceinline__ float pow2(int n) { return __uint_as_float((uint32_t)max(n + 127, 0) << 23); }

// max(a, |b|, |c|); a NaN counts for nothing.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
}

// Adds a part's sums v and (reference point, sum of weights) to a row's.
__device__ __forceinline__ void add_part(float& m, float& l, float (&o)[4], float2 ml, float4 v) {
  const float mn = fmaxf(m, ml.x), f0 = ex2_approx(m - mn), f = ex2_approx(ml.x - mn);
  m = mn;
  l = fmaf(l, f0, ml.y * f);
  o[0] = fmaf(o[0], f0, v.x * f), o[1] = fmaf(o[1], f0, v.y * f);
  o[2] = fmaf(o[2], f0, v.z * f), o[3] = fmaf(o[3], f0, v.w * f);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The shared memory of CTA `rank` of the cluster, by this CTA's address of the same place.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  return there;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_load1(uint32_t addr, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(addr, rank)) : "memory");
  return v;
}

// Two codes (one per 16-bit half, in bits 0-3) as f16 code - 8; HIGH: in bits 4-7, as 16 (code - 8).
template <bool HIGH>
__device__ __forceinline__ uint32_t codes_f16(uint32_t z) {
  const uint32_t x = (z & (HIGH ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
  return h2_bits(__hsub2(bits_h2(x), bits_h2(HIGH ? 0x64806480u : 0x64086408u)));
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                   : "r"(addr + 4 * i));
  }
}

// A lane's elements of a query row in shared memory: 32i + 8t .. + 7 of each block i.
template <int NB>
__device__ __forceinline__ void load_query(uint32_t row, int t, int dtype, float (&q)[NB][8]) {
#pragma unroll
  for (int i = 0; i < NB; i++) {
    uint32_t w[4];
    if (dtype == HCU_DT_F32) {
      lds_words<4>(row + (32 * i + 8 * t) * 4, w);
#pragma unroll
      for (int c = 0; c < 4; c++) q[i][c] = __uint_as_float(w[c]);
      lds_words<4>(row + (32 * i + 8 * t + 4) * 4, w);
#pragma unroll
      for (int c = 0; c < 4; c++) q[i][4 + c] = __uint_as_float(w[c]);
    } else {
      lds_words<4>(row + (32 * i + 8 * t) * 2, w);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const float2 h = f16x2_to_f2(w[c]);
        q[i][2 * c] = dtype == HCU_DT_F16 ? h.x : bf16_lo(w[c]);
        q[i][2 * c + 1] = dtype == HCU_DT_F16 ? h.y : bf16_hi(w[c]);
      }
    }
  }
}
__device__ __forceinline__ void store4_dt(void* p, size_t at, int dtype, const float (&x)[4]) {
  if (dtype == HCU_DT_F32) store4(static_cast<float*>(p) + at, x);
  else if (dtype == HCU_DT_F16) store4(static_cast<__half*>(p) + at, x);
  else store4(static_cast<__nv_bfloat16*>(p) + at, x);
}

constexpr int kMaxCluster = 8, kClusterChunks = 4;  // CTAs of a cluster, chunks of a warp in one at most
constexpr int kMaxParts = 320;  // CTAs of a call, and so of a unit
constexpr int STAGES = 2;
constexpr int paged_stage_bytes(int dh) { return CHUNK * (dh + dh / 8); }  // codes and scales, keys and values
constexpr int paged_row_floats(int dh) { return dh + 4; }  // of the warps' sums (a multiple of four)
constexpr size_t paged_smem(int dh, int rb) {
  return (size_t)NW * STAGES * paged_stage_bytes(dh) + (size_t)NW * rb * paged_row_floats(dh) * 4;
}
// Per SM.  One row per thread fits 128 registers; two (bf16, eight rows) do not: two CTAs 67 us, one 60 (32 sequences, 64 / 8 heads).
constexpr int paged_ctas(int dh, int ct) { return dh == 128 && ct == 2 ? 2 : 1; }

// The work of a call is a line of chunks: sequence after sequence, in each
// its KV heads, in each its row blocks, in each the chunks that hold visible tokens
// (one empty chunk where there are none: zeros are to be written).  CTA i of n
// takes the i-th of n equal pieces of the line and each of its warps an
// eighth of that, so a ragged batch and a single long sequence keep every warp
// busy to the end alike, and no warp waits for another before that.  A unit (a
// sequence's KV head and row block) that lies within a warp's piece is
// finished by that warp; the others leave records that are joined at the end.
struct PagedPlan {
  int total, share, more;  // chunks (below 2^31: the host checks); per CTA; the first `more` CTAs take one more
  int ctas;
  __device__ int start(int i) const { return i * share + min(i, more); }
  __device__ int cta_of(int x) const {
    const int edge = more * (share + 1);
    return x < edge ? x / (share + 1) : more + (x - edge) / share;
  }
};

// First token that a query at position pos sees (pos may be negative: pos + 1 - window could then pass int's range).
__device__ __forceinline__ int first_seen(int pos, int window) { return window > 0 && pos >= window ? pos + 1 - window : 0; }

// Chunk range of sequence b over all its queries: first chunk, count (at least 1).
__device__ __forceinline__ int2 paged_chunks(const PagedAttnArgs& a, int b) {
  int ctx = a.context[b];
  if (ctx > a.max_context || ctx < 0) ctx = 0;
  const int first = ctx - a.S;
  const int lo = first_seen(first, a.window);
  const int c_lo = lo / CHUNK, c_hi = (ctx + CHUNK - 1) / CHUNK;
  return make_int2(c_lo, max(1, c_hi - c_lo));
}

// A query (a weighted probability) is CT f16 numbers in as many columns, or MT
// in a column of MT products each; NC groups of eight columns make RB = 8 NC /
// CT rows per warp.  EXACT: code - 8 for both operands (f32 results), and the
// sums of 16 tokens are added in f32 outside of the tensor cores, whose own
// additions truncate: over 8192 tokens that came to 7e-6 of the result.
// Otherwise the codes as they are, the offset taken off the sums.
template <int DH, int CT, int MT, int NC, bool EXACT>
__global__ void __launch_bounds__(32 * NW, paged_ctas(DH, CT)) attn_paged_kernel(const PagedAttnArgs a) {
  constexpr int NB = DH / 32, ST = STAGES, SB = paged_stage_bytes(DH);
  constexpr int RG = 8 / CT, RB = RG * NC;      // rows per column group, per warp
  constexpr int NR = 2 / CT;                   // rows per thread and column group
  static_assert(CT * MT == 1 || (CT * MT == 2 && (MT == 1 || EXACT)), "one f16 number or two");
  constexpr bool WIDE = CT * MT == 2;          // two f16 numbers: queries may be f32
  constexpr int KB = CHUNK * DH / 2, CB = CHUNK * NB * 2;  // bytes of a stage's codes, of its scales
  // Steps of 16 tokens in the loop's body: with two of these the code outgrows the instruction cache (replayed graphs, bf16,
  // four tokens of 32 / 8 heads over 16 x 4000 tokens: 53.6 us unrolled, 50.2 rolled; f32, four tokens of 16 / 2 heads of 256
  // over 16 x 4096: 83 and 76; bf16, one token of 32 / 8 over 64 x 1612: 39.6 and 40.2).
  constexpr int kSteps = DH == 256 || NC == 2 ? 1 : 2;
  constexpr int RS = paged_row_floats(DH);
  constexpr size_t REC = (size_t)RB * (DH + 2);  // floats of a global record
  static_assert(RB * RS * 4 <= ST * SB, "a record fits a ring");
  static_assert(RB * DH * (WIDE ? 4 : 2) <= SB, "a segment's queries fit a stage");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float2 s_ml[RB];  // of the CTA's part (kCluster); s_mine: its sums
  __shared__ __align__(16) uint32_t s_mine;
  __shared__ int scan[NW], s_b, s_pos;
  // Records of a warp's units that lie only partly in its piece: [2w] the one that ends there, [2w + 1] the one that
  // goes on.  u0 < 0: none.
  __shared__ struct {
    int u0, n, b, kvh, rb, begins;
  } s_rec[2 * NW];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tok = (g >> 1) + 4 * (g & 1);  // token of accumulator row g (row g + 8: 8 more)

  // ---- this CTA's piece of the line ----
  const int per_chunk = a.kv.KV * a.nrb;  // units of a sequence, all of its chunk count
  PagedPlan plan;
  int seg_b, seg_base;  // sequence of the next segment, line position of its first chunk
  int pos, end, cta_first;
  if (a.split == kCluster) {
    const int unit = blockIdx.x / a.cluster, part = (blockIdx.x % a.cluster) * NW + warp, parts = a.cluster * NW;
    seg_b = unit / per_chunk, seg_base = 0;
    const int n = paged_chunks(a, seg_b).y;
    cta_first = (unit % per_chunk) * (n + kUnitCost) + kUnitCost;
    pos = cta_first + (int)((long long)n * part / parts), end = cta_first + (int)((long long)n * (part + 1) / parts);
    if (threadIdx.x < 2 * NW) s_rec[threadIdx.x].u0 = -1;
    __syncthreads();
  } else {
    // Every thread sums a run of sequences; the line position of each run follows from a scan.
    const int run = (a.batch + 32 * NW - 1) / (32 * NW), b0 = threadIdx.x * run, b1 = min(a.batch, b0 + run);
    int sum = 0;
    for (int b = b0; b < b1; b++) sum += paged_chunks(a, b).y + kUnitCost;
    int pre = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += x;
    }
    if (lane == 31) scan[warp] = pre;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      if (w < warp) pre += scan[w];
      total += scan[w];
    }
    plan.total = total * per_chunk;
    const int most = a.split == kLine ? (plan.total - 1) / a.min_chunks + 1 : (int)gridDim.x;
    plan.ctas = min((int)gridDim.x, most);
    plan.share = plan.total / plan.ctas;
    plan.more = plan.total % plan.ctas;
    if ((int)blockIdx.x >= plan.ctas) {
      if (a.split == kLine && threadIdx.x == 0) a.open[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    if (threadIdx.x < 2 * NW) s_rec[threadIdx.x].u0 = -1;
    if (a.split == kLine) {
      cta_first = plan.start(blockIdx.x);
      const int len = plan.start(blockIdx.x + 1) - cta_first, lo = (pre - sum) * per_chunk;
      if (cta_first >= lo && cta_first < pre * per_chunk) {  // one thread's run holds the first chunk
        int at = lo, b = b0;
        for (;; b++) {
          const int n = (paged_chunks(a, b).y + kUnitCost) * per_chunk;
          if (cta_first < at + n) break;
          at += n;
        }
        s_b = b;
        s_pos = at;
      }
      __syncthreads();
      seg_b = s_b;
      seg_base = s_pos;
      pos = cta_first + (int)((long long)len * warp / NW);
      end = cta_first + (int)((long long)len * (warp + 1) / NW);
    } else {  // whole units: every (gridDim.x * NW)-th
      __syncthreads();
      cta_first = 0;
      pos = blockIdx.x * NW + warp, end = a.batch * per_chunk;
      seg_b = 0, seg_base = 0;
    }
  }

  // The segment at line position `at` (or, unsplit, unit number `at`): chunks [c0, c1) of unit (b, kvh, rb), whose n
  // chunks begin at position u0, and the position behind it.  It may be empty (the position lies in a unit's cost).
  // seq_b and seq_base walk along.
  struct Segment {
    int b, kvh, rb, c0, c1, u0, n, next;
    bool begins, ends;
  };
  auto segment = [&](int at, int& seq_b, int& seq_base) -> Segment {
    Segment s;
    int u;
    int2 ch;
    if (a.split != kWarpUnits) {
      ch = paged_chunks(a, seq_b);
      while (at >= seq_base + (ch.y + kUnitCost) * per_chunk) {
        seq_base += (ch.y + kUnitCost) * per_chunk;
        ch = paged_chunks(a, ++seq_b);
      }
      s.b = seq_b;
      u = (at - seq_base) / (ch.y + kUnitCost);
      s.u0 = seq_base + u * (ch.y + kUnitCost) + kUnitCost;
      s.next = min(end, s.u0 + ch.y);
      s.c0 = ch.x + max(0, at - s.u0);
      s.c1 = ch.x + max(0, s.next - s.u0);
    } else {
      s.b = at / per_chunk;
      u = at % per_chunk;
      ch = paged_chunks(a, s.b);
      s.u0 = at;
      s.next = at + gridDim.x * NW;
      s.c0 = ch.x, s.c1 = ch.x + ch.y;
    }
    s.n = ch.y;
    s.begins = s.c0 == ch.x;
    s.ends = s.c1 == ch.x + ch.y;
    s.kvh = u / a.nrb, s.rb = u % a.nrb;
    return s;
  };

  // ---- this warp's ring: the chunks it will take, fetched ahead across segments ----
  const uint32_t ring = smem_u32(smem) + warp * ST * SB;
  float* buf = reinterpret_cast<float*>(smem + NW * ST * SB);  // [NW][RB][RS]: sums, M, l
  const int page_mask = (1 << a.kv.page_log2) - 1;
  int f_pos = pos, f_seq = seg_b, f_base = seg_base;  // the segment after the one being fetched
  Segment f{};
  int f_c = 0, f_lo, f_hi;
  const int32_t* f_table;
  // The tokens of a fetched sequence that any query sees, [f_lo, f_hi).
  auto fetch_seq = [&]() {
    int ctx = a.context[f.b];
    if (ctx > a.max_context || ctx < 0) ctx = 0;
    f_hi = ctx;
    f_lo = first_seen(ctx - a.S, a.window);
    f_table = a.table + (size_t)f.b * a.table_stride;
  };
  // The pages of chunk c's two halves of 16 tokens: -2 where no query sees a token of the half (not looked up), -1 for
  // every negative entry.
  auto look_up = [&](int c, int (&pg)[2]) {
#pragma unroll
    for (int p = 0; p < 2; p++) {
      const int t0 = c * CHUNK + 16 * p;
      pg[p] = c < f.c1 && t0 < f_hi && t0 + 16 > f_lo ? max(f_table[t0 >> a.kv.page_log2], -1) : -2;
    }
  };
  int f_page[2] = {-2, -2};
  auto enter = [&]() {  // the next segment with a chunk, from f_pos on
    do {
      f = segment(f_pos, f_seq, f_base);
      f_pos = f.next;
    } while (f.c0 >= f.c1 && f_pos < end);
    f_c = f.c0 < f.c1 ? f.c0 - 1 : f.c1;  // its queries come first
    fetch_seq();
  };
  if (pos < end) enter();
  // Fetches the next item, a segment's queries or a chunk, into a stage and looks the next chunk's pages up.  Returns
  // which halves of a chunk hold data.
  auto fetch = [&](int st) -> uint32_t {
    uint32_t halves = 0;
    const uint32_t dst = ring + st * SB;
    if (f_c < f.c0) {
      const int es = a.dtype == HCU_DT_F32 ? 4 : 2, ppr = DH * es / 16;  // 16-byte pieces of a row
      const int r0 = f.rb * RB;
#pragma unroll
      for (int i = 0; i < RB * DH * (WIDE ? 4 : 2) / 512; i++) {
        const int p = 32 * i + lane, r = p / ppr, rr = r0 + r;
        const bool there = r < RB && rr < a.R;
        const int sq = there ? rr / a.G : 0, h = f.kvh * a.G + (there ? rr % a.G : 0);
        const char* src = static_cast<const char*>(a.q) + (((size_t)f.b * a.S + sq) * a.H + h) * DH * es + (p % ppr) * 16;
        if (r < RB) copy16(dst + p * 16, src, there);
      }
      f_c++;
      look_up(f_c, f_page);
    } else if (f_c < f.c1) {
      if (a.kv.page_log2 >= 5 && (uint32_t)f_page[0] < (uint32_t)a.kv.n_pages && f_page[1] != -2) {
        // The whole chunk lies in one page: 32 rows in a piece.
        halves = 3u;
        const long long row = paged_row(a.kv, f_page[0], f.kvh, (f_c * CHUNK) & page_mask);
        const uint8_t* k = a.kv.k + row * (DH / 2) + lane * 16;
        const uint8_t* v = a.kv.v + row * (DH / 2) + lane * 16;
        const uint32_t d = dst + lane * 16;
#pragma unroll
        for (int i = 0; i < KB / 512; i++) {
          copy16(d + 512 * i, k + 512 * i);
          copy16(d + KB + 512 * i, v + 512 * i);
        }
#pragma unroll
        for (int i = 0; i < 2 * CB / 16; i += 32) {
          const int l = i + lane;
          copy16(dst + 2 * KB + l * 16, (l < CB / 16 ? a.kv.ks + l * 8 : a.kv.vs + (l - CB / 16) * 8) + row * NB);
        }
      } else {
        long long row[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
          const bool there = (uint32_t)f_page[p] < (uint32_t)a.kv.n_pages;
          if (!there && f_page[p] != -2 && lane == 0) atomicOr(a.status, HCU_DEVERR_BADARG);  // the table's entry is no page
          halves |= (there ? 1u : 0u) << p;
          row[p] = paged_row(a.kv, there ? f_page[p] : 0, f.kvh, (f_c * CHUNK + 16 * p) & page_mask);
        }
        const bool there[2] = {(halves & 1u) != 0, (halves & 2u) != 0};
#pragma unroll
        for (int p = 0; p < 2; p++) {
          const uint8_t* k = a.kv.k + row[p] * (DH / 2) + lane * 16;
          const uint8_t* v = a.kv.v + row[p] * (DH / 2) + lane * 16;
          const uint32_t d = dst + p * (KB / 2) + lane * 16;
#pragma unroll
          for (int i = 0; i < KB / 1024; i++) {
            copy16(d + 512 * i, k + 512 * i, there[p]);
            copy16(d + KB + 512 * i, v + 512 * i, there[p]);
          }
        }
        // scales: CB / 32 lanes per half, key scales then value scales
        constexpr int LH = CB / 32;
#pragma unroll
        for (int i = 0; i < 4 * LH; i += 32) {
          const int l = i + lane, p = (l / LH) & 1;
          const __half* src = (l / (2 * LH) ? a.kv.vs : a.kv.ks) + (p ? row[1] : row[0]) * NB + (l % LH) * 8;
          copy16(dst + 2 * KB + l * 16, src, p ? there[1] : there[0]);
        }
      }
      if (++f_c == f.c1 && f_pos < end) enter();
      look_up(f_c, f_page);
    }
    copy_commit();
    return halves;
  };
  uint32_t have = 0;  // two bits per stage
#pragma unroll
  for (int i = 0; i < ST; i++) have |= fetch(i) << (2 * i);
  int stage = 0;

  while (pos < end) {
    const Segment sg = segment(pos, seg_b, seg_base);
    const int b = sg.b, kvh = sg.kvh, rb = sg.rb, c1 = sg.c1;
    const bool begins = sg.begins, ends = sg.ends;
    pos = sg.next;
    if (sg.c0 >= c1) continue;
    const int r0 = rb * RB, rows = min(RB, a.R - r0);
    int ctx = a.context[b];
    if (ctx > a.max_context || ctx < 0) {
      if (lane == 0) atomicOr(a.status, HCU_DEVERR_BADARG);
      ctx = 0;
    }
    // The tokens that every row of this block sees: [lo_all, hi_all).
    const int pos_first = ctx - a.S + r0 / a.G, pos_last = ctx - a.S + (r0 + rows - 1) / a.G;
    const int lo_all = first_seen(pos_last, a.window), hi_all = max(0, pos_first + 1);
    // ---- query columns: column g of group nc is row / term of this lane's B fragments ----
    copy_wait<ST - 1>();
    __syncwarp();
    uint32_t qf[NC][MT][NB][4];
    float corr[NC][NB][NR];  // -8 sum(q) of the block (not EXACT), rows of this thread's accumulator columns 2t, 2t + 1
    float rs[NC][NR];        // score = rs * (kCodes * accumulated sum): together the factors can pass f32's range
    constexpr float kCodes = EXACT ? 1.f : 16777216.f;  // subnormal codes carry 2^-24
#pragma unroll
    for (int nc = 0; nc < NC; nc++) {
      const int r = nc * RG + (CT == 2 ? g >> 1 : g);
      float q[NB][8], top = 0.f;  // rows past the last are zeros
      load_query<NB>(ring + stage * SB + r * (DH * (a.dtype == HCU_DT_F32 ? 4 : 2)), t, a.dtype, q);
#pragma unroll
      for (int i = 0; i < NB; i++)
#pragma unroll
        for (int c = 0; c < 8; c++) top = fmaxf(top, fabsf(q[i][c]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^sq brings the row's largest magnitude into [2^13, 2^14)
      const int sq = top > 0.f ? max(-126, min(127, 140 - (int)(__float_as_uint(top) >> 23))) : 0;
      const float up = __uint_as_float((uint32_t)(sq + 127) << 23);
      const float back = ldexpf(a.scale_log2, -sq);
#pragma unroll
      for (int i = 0; i < NB; i++) {
        float sum = 0.f;
#pragma unroll
        for (int m = 0; m < 4; m++) {
          // register m: dimensions m and m + 4 of the lane's eight; odd m meets codes times 16
          __half o[2], low[2];
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float f = (m & 1) ? 0.0625f : 1.f;
            float v = q[i][m + 4 * c] * up;
            if (CT == 2 && (g & 1)) v -= __half2float(__float2half_rn(v));
            o[c] = __float2half_rn(v * f);
            if (MT == 2) low[c] = __float2half_rn((v - __half2float(__float2half_rn(v))) * f);
            if (!EXACT) sum += __half2float(o[c]) * ((m & 1) ? 16.f : 1.f);
          }
          qf[nc][0][i][m] = h2_bits(__halves2half2(o[0], o[1]));
          if (MT == 2) qf[nc][MT - 1][i][m] = h2_bits(__halves2half2(low[0], low[1]));
        }
        if (!EXACT) {
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          sum *= -8.f * 5.9604644775390625e-08f;  // -8 * 2^-24
          // column 2t is lane group g = 2t, column 2t + 1 the next
          const float u0 = __shfl_sync(0xffffffffu, sum, 8 * t), u1 = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
          corr[nc][i][0] = CT == 2 ? u0 + u1 : u0;
          if (NR == 2) corr[nc][i][NR - 1] = u1;
        }
      }
      rs[nc][0] = __shfl_sync(0xffffffffu, back, 8 * t);
      if (NR == 2) rs[nc][NR - 1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
    }

    __syncwarp();
    have = (have & ~(3u << (2 * stage))) | fetch(stage) << (2 * stage);
    stage ^= 1;

    float O[2 * NB][NC][4] = {};
    float M[NC][NR], L[NC][NR], E[NC][NR][NB];
#pragma unroll
    for (int nc = 0; nc < NC; nc++)
#pragma unroll
      for (int r = 0; r < NR; r++) {
        M[nc][r] = kNoM, L[nc][r] = 0.f;
#pragma unroll
        for (int i = 0; i < NB; i++) E[nc][r][i] = __uint_as_float(kMostE << 23);
      }

    for (int c = sg.c0; c < c1; c++) {
      copy_wait<ST - 1>();
      __syncwarp();
      const uint32_t st = ring + stage * SB;
      const uint32_t halves = (have >> (2 * stage)) & 3u;
      const int base = c * CHUNK;
      const bool whole = base >= lo_all && base + CHUNK <= hi_all && halves == 3u;
#pragma unroll kSteps
      for (int j = 0; j < 2; j++) {
        // ---- scores of 16 tokens ----
        float x[2][NC][NR];        // [accumulator row half][..]: score, log2 units
        uint32_t vsw[2][NB / 2];   // value scales of the thread's tokens, f16 pairs
        uint32_t kw[2][NB], ksw[2][NB / 2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const uint32_t row = 16 * j + 8 * u + tok;
          lds_words<NB>(st + row * (DH / 2) + t * NB * 4, kw[u]);
          lds_words<NB / 2>(st + 2 * KB + row * NB * 2, ksw[u]);
          lds_words<NB / 2>(st + 2 * KB + CB + row * NB * 2, vsw[u]);
#pragma unroll
          for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int r = 0; r < NR; r++) x[u][nc][r] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < NB; i++) {
          uint32_t a0[4], a1[4];
          const uint32_t w0 = kw[0][i] >> 8, w1 = kw[1][i] >> 8;
          if (EXACT) {
            a0[0] = codes_f16<false>(kw[0][i]), a0[1] = codes_f16<false>(kw[1][i]);
            a0[2] = codes_f16<true>(kw[0][i]), a0[3] = codes_f16<true>(kw[1][i]);
            a1[0] = codes_f16<false>(w0), a1[1] = codes_f16<false>(w1), a1[2] = codes_f16<true>(w0), a1[3] = codes_f16<true>(w1);
          } else {
            a0[0] = kw[0][i] & 0x000f000fu, a0[1] = kw[1][i] & 0x000f000fu;
            a0[2] = kw[0][i] & 0x00f000f0u, a0[3] = kw[1][i] & 0x00f000f0u;
            a1[0] = w0 & 0x000f000fu, a1[1] = w1 & 0x000f000fu, a1[2] = w0 & 0x00f000f0u, a1[3] = w1 & 0x00f000f0u;
          }
          float ks[2];
#pragma unroll
          for (int u = 0; u < 2; u++) ks[u] = (i & 1) ? f16x2_to_f2(ksw[u][i / 2]).y : f16x2_to_f2(ksw[u][i / 2]).x;
#pragma unroll
          for (int nc = 0; nc < NC; nc++) {
            float d[4];
            mma16816_zero(d, a0, qf[nc][0][i][0], qf[nc][0][i][1]);
            if (MT == 2) {
              float e[4];
              mma16816_zero(e, a0, qf[nc][MT - 1][i][0], qf[nc][MT - 1][i][1]);
              mma16816(d, a1, qf[nc][0][i][2], qf[nc][0][i][3]);
              mma16816(e, a1, qf[nc][MT - 1][i][2], qf[nc][MT - 1][i][3]);
              f2_get(f2_add(f2(d[0], d[1]), f2(e[0], e[1])), d[0], d[1]);
              f2_get(f2_add(f2(d[2], d[3]), f2(e[2], e[3])), d[2], d[3]);
            } else {
              mma16816(d, a1, qf[nc][0][i][2], qf[nc][0][i][3]);
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
              for (int r = 0; r < NR; r++) {
                float sum = d[2 * u + r];
                if (!EXACT) sum += corr[nc][i][r];
                if (CT == 2) sum += d[2 * u + 1];
                x[u][nc][r] = fmaf(ks[u], sum, x[u][nc][r]);
              }
            }
          }
        }
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < NR; r++) x[u][nc][r] = x[u][nc][r] * kCodes * rs[nc][r];
        if (!whole) {
          // Tokens outside a row's range and on missing pages weigh nothing; what their rows hold is not looked at.
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const int at = base + 16 * j + 8 * u + tok;
            const bool data = (halves >> j) & 1u;
            bool any = false;
#pragma unroll
            for (int nc = 0; nc < NC; nc++)
#pragma unroll
              for (int r = 0; r < NR; r++) {
                const int rl = nc * RG + t * NR + r, p = ctx - a.S + (r0 + rl) / a.G;
                const bool see = data && rl < rows && at <= p && at >= first_seen(p, a.window);
                x[u][nc][r] = see ? x[u][nc][r] : -INFINITY;
                any = any || see;
              }
            if (!any)
#pragma unroll
              for (int i = 0; i < NB / 2; i++) vsw[u][i] = 0u;
          }
        }
        // ---- probabilities, and weighted by the blocks' value scales ----
        float p[NC][2][NR] = {};
        auto weight = [&](int nc, int u, int r, int i2) {  // of two blocks, without E
          const float2 v = f16x2_to_f2(vsw[u][i2]);
          return f2_mul(f2(v.x, v.y), f2(p[nc][u][r], p[nc][u][r]));
        };
        uint64_t w[NC][2][NR][NB / 2];
        auto weigh = [&]() {
          float most = 0.f;
#pragma unroll
          for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
              for (int r = 0; r < NR; r++) {
                p[nc][u][r] = ex2_approx(x[u][nc][r] - M[nc][r]);
                most = fmaxf(most, p[nc][u][r]);
#pragma unroll
                for (int i2 = 0; i2 < NB / 2; i2++) {
                  w[nc][u][r][i2] = f2_mul(weight(nc, u, r, i2), f2(E[nc][r][2 * i2], E[nc][r][2 * i2 + 1]));
                  float w0, w1;
                  f2_get(w[nc][u][r][i2], w0, w1);
                  most = max_abs(most, w0, w1);
                }
              }
          // A token that one of the thread's rows sees and another does not: its scale, which may be NaN, is the first one's alone.
          if (NR * NC > 1 && !whole)
#pragma unroll
            for (int nc = 0; nc < NC; nc++)
#pragma unroll
              for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < NR; r++)
#pragma unroll
                  for (int i2 = 0; i2 < NB / 2; i2++) w[nc][u][r][i2] = x[u][nc][r] == -INFINITY ? 0 : w[nc][u][r][i2];
          return most;
        };
        if (__any_sync(0xffffffffu, weigh() > (float)(1 << kTop))) {
#pragma unroll
          for (int nc = 0; nc < NC; nc++)
#pragma unroll
            for (int r = 0; r < NR; r++) {
              float m = fmaxf(x[0][nc][r], x[1][nc][r]);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
              m = fmaxf(M[nc][r], ceilf(m));
              const int n = (int)fminf(m - M[nc][r], 300.f);  // whole: M moves by multiplying every E by 2^n, the sums stay
              M[nc][r] = m;
              L[nc][r] *= pow2(-n);
#pragma unroll
              for (int u = 0; u < 2; u++) p[nc][u][r] = ex2_approx(x[u][nc][r] - m);
#pragma unroll
              for (int i2 = 0; i2 < NB / 2; i2++) {
                float a0, a1, b0, b1;
                f2_get(x[0][nc][r] == -INFINITY ? 0 : weight(nc, 0, r, i2), a0, a1);
                f2_get(x[1][nc][r] == -INFINITY ? 0 : weight(nc, 1, r, i2), b0, b1);
                // the largest weights of both blocks, by their upper 16 bits
                uint32_t top = __byte_perm(__float_as_uint(fmaxf(fabsf(a0), fabsf(b0))), __float_as_uint(fmaxf(fabsf(a1), fabsf(b1))), 0x7632u);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
                for (int e = 0; e < 2; e++) {
                  const int i = 2 * i2 + e, big = (int)(top >> (16 * e + 7)) & 0xff;  // exponent bits
                  const int old = (int)(__float_as_uint(E[nc][r][i]) >> 23) + n;
                  const int now = min(min(old, (int)kMostE), 254 + kStart - big);  // the largest becomes 2^kStart, unless it is less
                  E[nc][r][i] = __uint_as_float((uint32_t)now << 23);
                  const float f = pow2(now - old);
#pragma unroll
                  for (int k = 0; k < 4; k++)
                    if (NR == 1 || (k & 1) == r) O[2 * i][nc][k] *= f, O[2 * i + 1][nc][k] *= f;
                }
              }
            }
          weigh();
        }
#pragma unroll
        for (int nc = 0; nc < NC; nc++)
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int r = 0; r < NR; r++) L[nc][r] += p[nc][u][r];
        // ---- values ----
        uint32_t vw[4][NB / 2];  // tokens t, t + 4, t + 8, t + 12: halfwords of the lane's dimensions
#pragma unroll
        for (int k = 0; k < 4; k++) lds_words<NB / 2>(st + KB + (16 * j + t + 4 * k) * (DH / 2) + g * NB * 2, vw[k]);
#pragma unroll
        for (int i2 = 0; i2 < NB / 2; i2++) {  // two blocks at a time
          uint32_t pb[2][NC][MT][2];  // [block] B fragments: tokens in pairs, column g
#pragma unroll
          for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int nc = 0; nc < NC; nc++) {
              float y[NR][2], l[NR][2];  // a weighted probability's first f16 number (exact in f32) and what is left
#pragma unroll
              for (int r = 0; r < NR; r++) {
                f2_get(w[nc][u][r][i2], y[r][0], y[r][1]);
                if (WIDE) {
                  y[r][0] = __uint_as_float(__float_as_uint(y[r][0]) & 0xffffe000u);
                  y[r][1] = __uint_as_float(__float_as_uint(y[r][1]) & 0xffffe000u);
                  f2_get(f2_fma(f2(y[r][0], y[r][1]), f2(-1.f, -1.f), w[nc][u][r][i2]), l[r][0], l[r][1]);
                }
              }
#pragma unroll
              for (int e = 0; e < 2; e++) {
                pb[e][nc][0][u] = movmatrix(h2_bits(CT == 2 ? __floats2half2_rn(y[0][e], l[0][e]) : __floats2half2_rn(y[0][e], y[NR - 1][e])));
                if (MT == 2) pb[e][nc][MT - 1][u] = movmatrix(h2_bits(__floats2half2_rn(l[0][e], l[NR - 1][e])));
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int i = 2 * i2 + e;
            const uint32_t sel = e ? 0x7632u : 0x5410u;
            uint32_t z0 = __byte_perm(vw[0][i2], vw[1][i2], sel), z1 = __byte_perm(vw[2][i2], vw[3][i2], sel);
#pragma unroll
            for (int m = 0; m < 2; m++) {
              if (EXACT) {
                const uint32_t av[4] = {codes_f16<false>(z0), codes_f16<true>(z0), codes_f16<false>(z1), codes_f16<true>(z1)};
#pragma unroll
                for (int nc = 0; nc < NC; nc++) {
                  float d[4];
                  mma16816_zero(d, av, pb[e][nc][MT - 1][0], pb[e][nc][MT - 1][1]);
                  if (MT == 2) mma16816(d, av, pb[e][nc][0][0], pb[e][nc][0][1]);
                  float(&o)[4] = O[2 * i + m][nc];
                  f2_get(f2_add(f2(o[0], o[1]), f2(d[0], d[1])), o[0], o[1]);
                  f2_get(f2_add(f2(o[2], o[3]), f2(d[2], d[3])), o[2], o[3]);
                }
              } else {
                // as the key codes, f16 subnormals; the offset is a product of its own
                const uint32_t av[4] = {z0 & 0x000f000fu, z0 & 0x00f000f0u, z1 & 0x000f000fu, z1 & 0x00f000f0u};
                const uint32_t off[4] = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};  // -8, -128 times 2^-24
#pragma unroll
                for (int nc = 0; nc < NC; nc++) {
                  mma16816(O[2 * i + m][nc], av, pb[e][nc][0][0], pb[e][nc][0][1]);
                  mma16816(O[2 * i + m][nc], off, pb[e][nc][0][0], pb[e][nc][0][1]);
                }
              }
              z0 >>= 8, z1 >>= 8;
            }
          }
        }
      }
      // ---- the stage is free for the chunk ST rounds on ----
      __syncwarp();
      have = (have & ~(3u << (2 * stage))) | fetch(stage) << (2 * stage);
      stage ^= 1;
    }

    // ---- the segment's sums ----
    const bool complete = begins && ends && a.split != kCluster;
    float* rec = ends ? buf + warp * RB * RS : reinterpret_cast<float*>(smem + warp * ST * SB);
#pragma unroll
    for (int nc = 0; nc < NC; nc++)
#pragma unroll
      for (int r = 0; r < NR; r++) {
        float l = L[nc][r];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int rl = nc * RG + t * NR + r;
        const float f = complete ? (l > 0.f ? kCodes / l : (l == 0.f ? 0.f : l)) : kCodes;  // no token: zeros; NaN stays
        float* row = rec + rl * RS;
#pragma unroll
        for (int i = 0; i < NB; i++) {  // dimensions 32i + 4g .. + 3
          const float *o0 = O[2 * i][nc], *o1 = O[2 * i + 1][nc];
          float4 v;
          const float fe = f * __uint_as_float((254u << 23) - __float_as_uint(E[nc][r][i]));  // f / E
          v.x = (CT == 2 ? o0[0] + o0[1] : o0[r]) * fe;
          v.y = (CT == 2 ? o0[2] + o0[3] : o0[2 + r]) * (0.0625f * fe);
          v.z = (CT == 2 ? o1[0] + o1[1] : o1[r]) * fe;
          v.w = (CT == 2 ? o1[2] + o1[3] : o1[2 + r]) * (0.0625f * fe);
          if (complete) {
            if (rl < rows) {
              const int rr = r0 + rl, s = rr / a.G, h = kvh * a.G + rr % a.G;
              const float y[4] = {v.x, v.y, v.z, v.w};
              store4_dt(a.out, (((size_t)b * a.S + s) * a.H + h) * DH + 32 * i + 4 * g, a.dtype, y);
            }
          } else {
            *reinterpret_cast<float4*>(row + 32 * i + 4 * g) = v;
          }
        }
        if (!complete && g == 0) row[DH] = M[nc][r], row[DH + 1] = l;
      }
    if (!complete && lane == 0) {
      auto& i = s_rec[2 * warp + (ends ? 0 : 1)];
      i.u0 = sg.u0, i.n = sg.n, i.b = b, i.kvh = kvh, i.rb = rb, i.begins = begins;
    }
  }
  __syncthreads();

  // ---- join the records: neighbours of the same unit ----
  auto finish = [&](const float (&o)[4], float l, int b, int kvh, int rr, int d) {
    const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const float y[4] = {o[0] * f, o[1] * f, o[2] * f, o[3] * f};
    const int s = rr / a.G, h = kvh * a.G + rr % a.G;
    store4_dt(a.out, (((size_t)b * a.S + s) * a.H + h) * DH + d, a.dtype, y);
  };
  constexpr int TPE = DH / 4;  // threads that hold a row
  if (a.split == kCluster) {
    // The CTA's parts go into one, in the place of the first; then every CTA of the cluster joins a share of the outputs.
    const int unit = blockIdx.x / a.cluster, b = unit / per_chunk, kvh = unit % per_chunk / a.nrb, rb = unit % per_chunk % a.nrb;
    const int r0 = rb * RB, rows = min(RB, a.R - r0);
    uint32_t members = 0;
    for (int k = 0; k < 2 * NW; k++) members |= (s_rec[k].u0 >= 0 ? 1u : 0u) << k;
    auto record = [&](int w) { return (w & 1) ? reinterpret_cast<float*>(smem + (w >> 1) * ST * SB) : buf + (w >> 1) * RB * RS; };
    float* mine = record(members ? __ffs(members) - 1 : 0);
    for (int i = threadIdx.x; i < rows * TPE; i += 32 * NW) {
      const int r = i / TPE, d = 4 * (i % TPE);
      float m = kNoM, l = 0.f, o[4] = {};
#pragma unroll 1
      for (uint32_t x = members; x; x &= x - 1) {
        const float* rec = record(__ffs(x) - 1) + r * RS;
        add_part(m, l, o, *reinterpret_cast<const float2*>(rec + DH), *reinterpret_cast<const float4*>(rec + d));
      }
      *reinterpret_cast<float4*>(mine + r * RS + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) s_ml[r] = make_float2(m, l);
    }
    if (threadIdx.x == 0) s_mine = smem_u32(mine);
    cluster_sync();
    const int share = a.cluster * 32 * NW;
    for (int i = (blockIdx.x % a.cluster) * 32 * NW + threadIdx.x; i < rows * TPE; i += share) {
      const int r = i / TPE, d = 4 * (i % TPE);
      float m = kNoM, l = 0.f, o[4] = {};
#pragma unroll 1
      for (int c = 0; c < a.cluster; c++) {
        const float2 ml = cluster_load2(smem_u32(&s_ml[r]), c);
        if (ml.y == 0.f) continue;  // no token: the place may hold anything
        add_part(m, l, o, ml, cluster_load4(cluster_load1(smem_u32(&s_mine), c) + (r * RS + d) * 4, c));
      }
      finish(o, l, b, kvh, r0 + r, d);
    }
    cluster_sync();  // the others' reads of this CTA's shared memory are done
    return;
  }
  int4 open = make_int4(0, 0, 0, 0);
  for (int k = 0; k < 2 * NW;) {
    const int u0 = s_rec[k].u0;
    if (u0 < 0) {
      k++;
      continue;
    }
    const int first = k;
    int last = k;
    uint32_t members = 0;
    for (; k < 2 * NW && (s_rec[k].u0 == u0 || s_rec[k].u0 < 0); k++)
      if (s_rec[k].u0 == u0) members |= 1u << k, last = k;
    const int b = s_rec[first].b, kvh = s_rec[first].kvh, rb = s_rec[first].rb;
    const bool whole = s_rec[first].begins && !(last & 1);  // no other CTA has a part of the unit
    const int r0 = rb * RB, rows = min(RB, a.R - r0);
    // The unit's first CTA leaves its part in its second record, the others in their first.
    float* mine = a.part + ((size_t)blockIdx.x * 2 + (u0 >= cta_first ? 1 : 0)) * REC;
    for (int i = threadIdx.x; i < rows * TPE; i += 32 * NW) {
      const int r = i / TPE, d = 4 * (i % TPE);
      float m = kNoM, l = 0.f, o[4] = {};
#pragma unroll 1
      for (uint32_t x = members; x; x &= x - 1) {
        const int w = __ffs(x) - 1;
        const float* rec = ((w & 1) ? reinterpret_cast<const float*>(smem + (w >> 1) * ST * SB) : buf + (w >> 1) * RB * RS) + r * RS;
        const float2 ml = *reinterpret_cast<const float2*>(rec + DH);
        const float4 v = *reinterpret_cast<const float4*>(rec + d);
        add_part(m, l, o, ml, v);
      }
      if (whole) {
        finish(o, l, b, kvh, r0 + r, d);
      } else {
        *reinterpret_cast<float4*>(mine + r * DH + d) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0) *reinterpret_cast<float2*>(mine + RB * DH + 2 * r) = make_float2(m, l);
      }
    }
    if (!whole && u0 >= cta_first)
      open = make_int4(plan.cta_of(u0 + s_rec[first].n - 1) - (int)blockIdx.x + 1, b, kvh, rb);
  }
  if (a.split == kLine && threadIdx.x == 0) a.open[blockIdx.x] = open;
}

// Joins the parts of the units that several CTAs share: block (c, r) row r of
// the unit that begins in CTA c and goes on in the CTAs behind it.  It starts
// while the CTAs above end and waits for all of them (programmatic dependent
// launch): joining by the last CTA to arrive instead cost a fence, an atomic
// and a serial walk, 13 us against 4 us behind the last CTA of one sequence of
// 131072 keys.
template <int DH, int RB>
__global__ void __launch_bounds__(128) attn_paged_join_kernel(const PagedAttnArgs a) {
  constexpr size_t REC = (size_t)RB * (DH + 2);
  constexpr int TPE = DH / 4, GROUPS = 128 / TPE;  // threads that hold a row, groups that share the parts
  __shared__ float w[kMaxParts], red[8];
  __shared__ __align__(16) float sums[GROUPS][DH];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.y;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 open = a.open[blockIdx.x];
  const int n_parts = open.x, rr = open.w * RB + r;
  if (n_parts == 0 || rr >= a.R) return;
  // the unit's first CTA left its part in its second record, the others in their first
  auto record = [&](int i) { return a.part + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * REC; };
  float m = kNoM, l = 0.f;
  for (int i = tid; i < n_parts; i += 128) {
    const float2 ml = *reinterpret_cast<const float2*>(record(i) + RB * DH + 2 * r);
    const float mn = fmaxf(m, ml.x);
    l = fmaf(l, ex2_approx(m - mn), ml.y * ex2_approx(ml.x - mn));
    m = mn;
    w[i] = ml.x;
  }
  const float top = warp_max(m);
  if (lane == 0) red[warp] = top;
  __syncthreads();
  const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  l = warp_sum(l * ex2_approx(m - M));
  if (lane == 0) red[4 + warp] = l;
  const int grp = tid / TPE, d = 4 * (tid % TPE);
  float o[4] = {};
  for (int p0 = grp; p0 < n_parts; p0 += 8 * GROUPS) {
    float4 v[8];
#pragma unroll
    for (int c = 0; c < 8; c++)
      v[c] = *reinterpret_cast<const float4*>(record(min(p0 + c * GROUPS, n_parts - 1)) + r * DH + d);
#pragma unroll
    for (int c = 0; c < 8; c++) {
      const float f = p0 + c * GROUPS < n_parts ? ex2_approx(w[p0 + c * GROUPS] - M) : 0.f;
      if (p0 + c * GROUPS < n_parts)
        o[0] = fmaf(v[c].x, f, o[0]), o[1] = fmaf(v[c].y, f, o[1]), o[2] = fmaf(v[c].z, f, o[2]), o[3] = fmaf(v[c].w, f, o[3]);
    }
  }
  *reinterpret_cast<float4*>(&sums[grp][d]) = make_float4(o[0], o[1], o[2], o[3]);
  __syncthreads();
  if (grp != 0) return;
  l = (red[4] + red[5]) + (red[6] + red[7]);
  const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no token: zeros; NaN stays
  float y[4];
#pragma unroll
  for (int c = 0; c < 4; c++) {
    y[c] = 0.f;
#pragma unroll
    for (int k = 0; k < GROUPS; k++) y[c] += sums[k][d + c];
    y[c] *= f;
  }
  const int s = rr / a.G, h = open.z * a.G + rr % a.G;
  store4_dt(a.out, (((size_t)open.y * a.S + s) * a.H + h) * DH + d, a.dtype, y);
}

template <int DH, int CT, int MT, int NC, bool EXACT>
int launch(hcu_context* h, PagedAttnArgs a) {
  const char* op = "hcu_attention_paged";
  constexpr int RB = 8 * NC / CT;
  constexpr size_t smem = paged_smem(DH, RB), record = (size_t)RB * (DH + 2) * sizeof(float);
  auto kern = attn_paged_kernel<DH, CT, MT, NC, EXACT>;
  static std::atomic<uint64_t> attr_done{0};  // per device
  HCU_TRY(once_per_device(attr_done, h->device, [&]() -> int {
    return check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), op);
  }));
  static_assert(smem <= (size_t)(227 * 1024), "shared memory");
  a.nrb = (a.R + RB - 1) / RB;
  const long long units = (long long)a.batch * a.kv.KV * a.nrb;
  if (units > 0x7fffffffLL) return fail(HCU_EINVAL, "%s: batch x KV x query row blocks too large", op);
  long long grid = std::min(kMaxParts, h->sm_count * paged_ctas(DH, CT));
  // The line must not pass 2^31 and the records must fit the workspace (behind the other ops' tickets).
  const size_t room = h->workspace_bytes > kTicketBytes ? h->workspace_bytes - kTicketBytes : 0;
  const long long span = a.window > 0 ? std::min<long long>(a.max_context, (long long)a.window + a.S + CHUNK) : a.max_context;
  const long long most = units * (span / CHUNK + 2 + kUnitCost);  // chunks
  a.min_chunks = h->opt_attn_chunk > 0 ? (int)std::min<int64_t>(1 << 24, (h->opt_attn_chunk + CHUNK - 1) / CHUNK) : 8;
  // A cluster's CTAs, as many as there are chunks for their warps and slots for all.
  const long long chunks = (span + CHUNK - 1) / CHUNK + (a.window > 0 ? 1 : 0);
  a.cluster = 1;
  while (a.cluster < kMaxCluster && a.cluster * NW < chunks && 2 * a.cluster * units <= grid) a.cluster *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(32 * NW);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = h->stream;
  cfg.attrs = attr;
  if (chunks <= std::min(kMaxCluster, kClusterChunks * a.cluster) * NW && units <= grid && h->opt_attn_chunk == 0) {
    a.split = kCluster;
    cfg.gridDim = dim3((unsigned)(units * a.cluster));
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess) return HCU_OK;
    (void)cudaGetLastError();  // no room for a cluster on this device: by the other ways
  }
  if (room >= (size_t)grid * (2 * record + sizeof(int4)) && most < 0x7fffffffLL) {
    a.split = kLine;
    grid = std::min(grid, (most + a.min_chunks - 1) / a.min_chunks);
  } else {
    a.split = kWarpUnits;
    grid = std::min(grid, (units + NW - 1) / NW);
  }
  a.open = reinterpret_cast<int4*>(static_cast<uint8_t*>(h->workspace) + kTicketBytes);
  a.part = reinterpret_cast<float*>(a.open + grid);
  cfg.gridDim = dim3((unsigned)grid);
  cfg.numAttrs = 0;
  (void)cudaLaunchKernelEx(&cfg, kern, a);
  HCU_TRY(after_launch("hcu_attention_paged: launch"));  // takes the error, if there is one, so that no later call finds it
  if (a.split != kLine || grid == 1) return HCU_OK;
  cfg.gridDim = dim3((unsigned)(grid - 1), RB);  // no unit goes on behind the last CTA
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  (void)cudaLaunchKernelEx(&cfg, attn_paged_join_kernel<DH, RB>, a);
  return after_launch("hcu_attention_paged: join");
}

template <int DH>
int launch_dh(hcu_context* h, const PagedAttnArgs& a) {
  if (a.dtype == HCU_DT_BF16) {
    // One f16 number per query where the rows need the columns: its rounding (2^-11) is below the result's (2^-8).
    if (a.R <= 4) return launch<DH, 2, 1, 1, false>(h, a);
    if constexpr (DH == 128)
      if (a.R > 8) return launch<DH, 1, 1, 2, false>(h, a);
    return launch<DH, 1, 1, 1, false>(h, a);
  }
  if (a.dtype == HCU_DT_F16 && a.R <= 4) return launch<DH, 2, 1, 1, false>(h, a);
  if (a.R > 4) return launch<DH, 1, 2, 1, true>(h, a);
  return launch<DH, 2, 1, 1, true>(h, a);
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
  if (!q || !out || (!p->block_table && p->max_context) || !p->context) return fail(HCU_EINVAL, "%s: null argument", op);
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
  a.batch = (int)p->batch;
  return kv->Dh == 128 ? hcu::launch_dh<128>(h, a) : hcu::launch_dh<256>(h, a);
}
