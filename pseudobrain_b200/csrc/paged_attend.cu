// Attention of one new token per sequence over the paged cache.
//
// The work is cut into units of 16 entries of one (sequence, key head, row tile): a row tile is
// up to 16 of the query heads that share the key head. All units of a launch stand in one line
// (sequence by sequence, head by head, entry by entry) and every warp of the grid takes an equal
// run of it, so ragged lengths, one long sequence and many short ones load the SMs alike. A warp
// walks its run with an online softmax (base 2) and writes a head's result when its run holds
// the whole head, else the partial (maximum, sum, weighted values) of its piece; the join
// kernel, launched behind it, merges the pieces of each head and, when asked, turns the scores
// kept in the workspace into weights and adds them to the cache's mass. Few heads of moderate
// length take the other way: a cluster of 1 to 8 CTAs per head, whose warps share its units and
// join through distributed shared memory, one launch in all (see `head_cluster`).
#include <atomic>

#include "common.cuh"
#include "paged.cuh"
#include "tc.cuh"
#include "tma_host.h"

namespace pbk {
namespace {

constexpr int kUnit = 16;           // entries per unit
constexpr int kRing = 192 * 1024;   // staging bytes per CTA
constexpr int kMinUnits = 2;        // units per warp below which fewer warps take part
constexpr int kClusterUnits = 320;  // most units per CTA where a cluster takes a whole head
constexpr int kMassThreads = 256;
constexpr int kPad = 4;             // floats after a partial row's D values: maximum, sum, two unused

template <int D>
struct Shape {
  static constexpr int kWarps = D == 256 ? 6 : 8;
  static constexpr int kTile = kUnit * D * 2;  // bytes of a unit's keys (or values)
  static constexpr int kStages = kRing / (kWarps * 2 * kTile);
};

struct AttendArgs {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  int batch, width, page, log_page;
  int kv, groups, rt, rows;  // key heads, query heads per key head, row tiles, rows per tile
  int window, sinks, accumulate;
  float scale_log2, offset;  // offset: see `finite`
  const uint16_t* q;
  int64_t q_sb, q_sh;
  void* out;
  int64_t out_sb, out_sh;
  int out_f32;
  float* lse;                // [batch, h], natural logarithm
  float* mass;
  int64_t meta_page, meta_head;
  int pages;
  // workspace
  int64_t* base;             // [batch + 1] units of the sequences before, per (head, row tile)
  int4* open;                // [runs] the head that a run begins and does not end: its sequence (-1:
                             // none), its index among the sequence's heads and row tiles, the run that ends it
  float* part;               // [runs][2][rows][D + kPad]
  float* lse2;               // [batch, h] base 2
  float* scores;             // [units][rows][16] base 2
  int64_t whole_units;       // score units set apart per head where a CTA takes a whole head
  int* err;
};

// A maximum over no scores (or over -inf alone) as 0: 2^(-inf - 0) is then 0 without a branch,
// and a NaN score stays NaN. Weights are 2^(score - finite(max) + offset): fp16 weights are kept
// 2^14 above their value, so that an entry 2^-38 below the heaviest still counts (fp16 ends at
// 2^-24, and a long cache may hold 10^6 such entries); bf16 has fp32's range and needs none.
__device__ __forceinline__ float finite(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool F16>
__device__ __forceinline__ float round16(float x) {
  return F16 ? __half2float(__float2half_rn(x)) : __bfloat162float(__float2bfloat16_rn(x));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// Keys and values are read once per step and layer: marked to leave L2 first, they pass through
// it beside the scores and masses that are read again at the launch's end (ragged batch of 64,
// 1.04 GB with weights: 211 -> 204 us; without weights 184 -> 180).
__device__ __forceinline__ uint64_t streaming_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w, int v, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(tc::smem_u32(dst)),
      "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "l"(policy)
      : "memory");
}

// The units of one sequence: the sinks' units that lie before the window's, then those from the
// window's first entry on.
struct Span {
  int n, lo, sink_units, first, units;  // entries; first entry of the window; ...; first window unit; all units
  __device__ Span() {}
  __device__ Span(const AttendArgs& a, int b) {
    n = paged::clamp_length(a.lengths[b], a.width, a.page);
    lo = a.window > 0 ? max(0, n - a.window) : 0;
    first = lo / kUnit;
    sink_units = a.sinks >= lo ? first : min((a.sinks + kUnit - 1) / kUnit, first);
    units = sink_units + (n + kUnit - 1) / kUnit - first;
  }
  __device__ int entry(int t) const { return (t < sink_units ? t : first + t - sink_units) * kUnit; }
};

// Units per run: equal for all but the last run, at least kMinUnits.
__device__ __forceinline__ int run_length(int64_t total, int warps) {
  const int64_t x = total + warps - 1;
  const int64_t len = (x >> 32) == 0 ? (uint32_t)x / (uint32_t)warps : x / warps;
  return max((int)len, kMinUnits);
}
// The run that holds unit u.
__device__ __forceinline__ int run_of(int64_t u, int length) {
  return (u >> 32) == 0 ? (int)((uint32_t)u / (uint32_t)length) : (int)(u / length);
}

constexpr float kLn2 = 0.6931471805599453f;

// The sum over the 8 lanes that hold a query row's entries.
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

template <bool F16>
__device__ __forceinline__ void store_out(const AttendArgs& a, int64_t at, float y) {
  if (a.out_f32) static_cast<float*>(a.out)[at] = y;
  else if (F16) static_cast<__half*>(a.out)[at] = __float2half_rn(y);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
}

// The mass of quarter i (four entries; i / 4 counts the head's units) of one (sequence, key
// head): one page id and one 16-byte access serve the four. Loaded apart from the addition, so
// that it is on its way while the rows' logarithms are still being joined.
struct Quarter {
  float4* to = nullptr;  // nullptr: past the length, or on a page outside the pool
  float4 have;
  int left;              // entries of the sequence from the quarter's first on
  __device__ Quarter() {}
  __device__ Quarter(const AttendArgs& a, int b, int h, const Span& s, int i) {
    const int e = s.entry(i / 4) + i % 4 * 4;
    left = s.n - e;
    if (left <= 0) return;
    const int page = paged::page_of(a.table + b * a.table_stride, e, a.log_page, a.pages);
    if (page < 0) return;
    to = reinterpret_cast<float4*>(a.mass + page * a.meta_page + h * a.meta_head + (e & (a.page - 1)));
    have = *to;
  }
  // Adds the quarter's weights. `scores` are those of the head's first unit in the first row tile,
  // `tile` floats from one row tile's to the next's; lse2[r] the rows' logarithms (INFINITY for a
  // row without weight: it adds 0).
  __device__ void add(const AttendArgs& a, int i, const float* scores, int64_t tile, const float* lse2) const {
    if (to == nullptr) return;
    const float* x = scores + (int64_t)(i / 4) * (kUnit * a.rows) + i % 4 * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r0 = 0; r0 < a.groups; r0 += a.rows, x += tile) {
      const int rows = min(a.rows, a.groups - r0);
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const float4 y = *reinterpret_cast<const float4*>(x + r * kUnit);
        const float l = lse2[r0 + r];
        sum.x += ex2(y.x - l), sum.y += ex2(y.y - l), sum.z += ex2(y.z - l), sum.w += ex2(y.w - l);
      }
    }
    if (left >= 4) {
      *to = make_float4(have.x + sum.x, have.y + sum.y, have.z + sum.z, have.w + sum.w);
    } else {  // the sequence's last entries; rows past them are left alone
      float* f = reinterpret_cast<float*>(to);
      f[0] = have.x + sum.x;
      if (left > 1) f[1] = have.y + sum.y;
      if (left > 2) f[2] = have.z + sum.z;
    }
  }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t x;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t x;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of CTA `rank`'s shared memory, at the place that `p` has in this CTA's.
__device__ __forceinline__ float remote(const float* p, uint32_t rank) {
  uint32_t at;
  float x;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(tc::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}

// Keys are the M of both products and the query rows their N: S^T = K Q^T (A = 16 keys by
// ldmatrix, B = Q^T in registers) and O^T += V^T P^T (A = V^T by ldmatrix.trans, B = P^T from
// S^T's accumulators by two 8 x 8 transposes). With at most 16 rows the tcgen05 shapes would
// run at a sixteenth of their width, and at HBM's pace (23 bytes per clock and SM) these
// instructions are idle most of the time: the kernel is bound by the bytes of K and V.
//
// Staging: each warp owns a ring of kStages units filled by TMA (a box of 16 rows of 64
// elements per 128 bytes of the head, one per 8 rows when pages hold 8), 128-byte swizzled so
// that ldmatrix reads are free of conflicts, and refills a stage as soon as it has read it. No
// barrier between warps inside the loop. The ring's 192 KB in flight per SM cover the latency
// at full bandwidth several times over; the next unit's page id is read a unit ahead.
//
// Each unit's product with V starts from zero and is added to the running result by fp32 fma's. The
// tensor cores truncate what they add to an accumulator: with the running result kept there, heads
// of 131072 entries in one run each lost 3e-4 of the result (values of 1; 5e-4 at a mean of 0.5),
// always towards zero; now that is 1e-5 at most, and nothing got slower but heads of 256 with more
// than 8 rows (24 x 4 x 8000 entries, 16 rows: 106 -> 116 us in bf16, 105 -> 107 in fp16).
//
// Weights enter the product with V as two 16-bit numbers, the rounded weight and what the
// rounding left (16 bits together in bf16, 22 in fp16), so that a 16-bit result's own rounding is
// the largest error. The second product runs in the tensor cores' idle time where there are at most
// 8 rows and the heads are no longer than 128; fp16 heads of 256 pay for it (window case 54.7 ->
// 57.9 us, 24 x 4 x 8000 entries of 16 rows 107 -> 114).
template <int D, int NT, bool F16, bool WHOLE>
__global__ void __launch_bounds__(32 * Shape<D>::kWarps, 1)
    paged_attend_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                        const AttendArgs a) {
  using S = Shape<D>;
  constexpr int kK = D / 16;
  constexpr int kThreads = 32 * S::kWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t s_full[S::kWarps][S::kStages];
  __shared__ int64_t s_sum[S::kWarps], s_off[S::kWarps];
  __shared__ int s_seq[S::kWarps];
  __shared__ float2 s_ml[WHOLE ? S::kWarps : 1][16], s_joined[16];  // WHOLE: (maximum, sum) per row
  __shared__ float s_lse[16];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nwarps = gridDim.x * S::kWarps;
  const int pairs = a.kv * a.rt;  // (key head, row tile) of a sequence
  const uint32_t rank = WHOLE ? cluster_rank() : 0, ctas = WHOLE ? cluster_size() : 1;
  paged::launch_next();
  if (tid == 0) {
    tc::prefetch_tmap(&mk);
    tc::prefetch_tmap(&mv);
  }

  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) tc::mbar_init(&s_full[warp][i], 1);
    tc::fence_barrier_init();
  }
  __syncwarp();
  paged::wait_previous();

  struct Walk {
    int b, pair, t;
    Span s;
  };
  Walk c;
  int64_t u0 = 0;  // the run's first unit in the line (WHOLE: among the scores set apart)
  int run = 0, length = 0, count;
  if (WHOLE) {
    const int head = blockIdx.x / ctas, part = rank * S::kWarps + warp, parts = ctas * S::kWarps;
    c.b = head / pairs;
    c.pair = head % pairs;
    c.s = Span(a, c.b);
    c.t = (int)((int64_t)c.s.units * part / parts);
    count = (int)((int64_t)c.s.units * (part + 1) / parts) - c.t;
    u0 = head * a.whole_units + c.t;
  } else {
    // ---- where each warp's run starts: a scan of the sequences' units by the whole CTA
    const int per = (a.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += Span(a, b).units;
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += x;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    before -= mine;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w];
    }
    length = run_length(total * pairs, nwarps);
    int64_t at = before;
    for (int b = b0; b < b1; ++b) {
      const Span s(a, b);
      if (blockIdx.x == 0) a.base[b] = at;
      const int64_t from = at * pairs, to = from + (int64_t)s.units * pairs;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const int64_t u = (int64_t)(w * gridDim.x + blockIdx.x) * length;
        if (u >= from && u < to) s_seq[w] = b, s_off[w] = u - from;
      }
      at += s.units;
    }
    if (blockIdx.x == 0 && tid == 0) a.base[a.batch] = total;
    __syncthreads();
    run = warp * gridDim.x + blockIdx.x;  // neighbouring runs on different SMs
    u0 = (int64_t)run * length;
    count = (int)max((int64_t)0, min((int64_t)length, total * pairs - u0));
    if (lane == 0) a.open[run] = make_int4(-1, 0, 0, 0);
    if (count == 0) return;
    c.b = s_seq[warp];
    c.s = Span(a, c.b);
    c.pair = run_of(s_off[warp], c.s.units);
    c.t = (int)(s_off[warp] - (int64_t)c.pair * c.s.units);
  }

  // ---- the producer's position (p) runs ahead of the consumer's (c)
  Walk p = c;
  auto advance = [&](Walk& w) {
    if (++w.t < w.s.units || WHOLE) return;
    w.t = 0;
    if (++w.pair < pairs) return;
    w.pair = 0;
    do {
      if (++w.b >= a.batch) return;
      w.s = Span(a, w.b);
    } while (w.s.units == 0);
  };
  const bool small = a.page < kUnit;  // pages of 8: two per unit
  auto page_ids = [&](const Walk& w) {
    if (w.b >= a.batch || w.t >= w.s.units) return make_int2(-1, -1);
    const int32_t* row = a.table + w.b * a.table_stride;
    const int i = w.s.entry(w.t) >> a.log_page;
    return make_int2(row[i], small && i + 1 < a.width ? row[i + 1] : -1);
  };
  const uint64_t policy = streaming_policy();
  uint8_t* my_ring = ring + warp * S::kStages * 2 * S::kTile;
  auto issue = [&](const Walk& w, int2 ids, int stage) {
    if (lane == 0) {
      uint64_t* bar = &s_full[warp][stage];
      uint8_t* k = my_ring + stage * 2 * S::kTile;
      uint8_t* v = k + S::kTile;
      const int h = w.pair / a.rt, row = w.s.entry(w.t) & (a.page - 1);
      tc::mbar_expect_tx(bar, 2 * S::kTile);
      tma_load_5d(k, &mk, bar, 0, row, 0, h, ids.x, policy);
      tma_load_5d(v, &mv, bar, 0, row, 0, h, ids.x, policy);
      if (small) {
        tma_load_5d(k + S::kTile / 2, &mk, bar, 0, 0, 0, h, ids.y, policy);
        tma_load_5d(v + S::kTile / 2, &mv, bar, 0, 0, 0, h, ids.y, policy);
      }
    }
  };
  int2 ids = page_ids(p);
  const int ahead = min(S::kStages, count);
  for (int i = 0; i < ahead; ++i) {
    issue(p, ids, i);
    advance(p);
    ids = page_ids(p);
  }

  // 16-byte chunk ch of entry r in a staged unit: 8-row blocks of 1 KB per 64 elements
  const uint32_t block8 = small ? (D / 64) * 1024u : 1024u, block64 = small ? 1024u : 2048u;
  auto at = [&](int r, int ch) {
    return (r >> 3) * block8 + (ch >> 3) * block64 + (r & 7) * 128u + (((ch & 7) ^ (r & 7)) << 4);
  };
  const int g = lane >> 2, t4 = lane & 3, mi = lane >> 3;

  uint32_t qb[NT][kK][2];
  float o[NT][kK][4];
  float m[NT][2], l[NT][2];
  if (WHOLE) {  // a warp without units joins an empty part
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int kk = 0; kk < kK; ++kk) o[nt][kk][0] = o[nt][kk][1] = o[nt][kk][2] = o[nt][kk][3] = 0.f;
  }
  int rows = min(a.rows, a.groups);
  bool fresh = true, ok = true;
  int begun = c.t;  // first unit of the current piece in its head
  int stage = 0;
  uint32_t parity = 0;

  int i = 0;
  for (; i < count; ++i) {
    const int h = c.pair / a.rt, r0 = (c.pair % a.rt) * a.rows;
    if (fresh) {
      fresh = false;
      begun = c.t;
      rows = min(a.rows, a.groups - r0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool has = 8 * nt + g < rows;
        const uint16_t* qr = a.q + c.b * a.q_sb + (int64_t)(h * a.groups + r0 + 8 * nt + g) * a.q_sh;
#pragma unroll
        for (int kk = 0; kk < kK; ++kk) {
          qb[nt][kk][0] = has ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 2 * t4) : 0u;
          qb[nt][kk][1] = has ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8 + 2 * t4) : 0u;
          o[nt][kk][0] = o[nt][kk][1] = o[nt][kk][2] = o[nt][kk][3] = 0.f;
        }
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
    }
    if (!__all_sync(0xffffffffu, tc::mbar_wait(&s_full[warp][stage], parity))) {
      if (lane == 0 && a.err) atomicCAS(a.err, 0, 401);
      ok = false;
      break;
    }
    uint8_t* stage_k = my_ring + stage * 2 * S::kTile;
    const uint32_t kb = tc::smem_u32(stage_k), vb = kb + S::kTile;

    float sc[NT][4], sd[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = sd[nt][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < kK; ++kk) {
      uint32_t x0, x1, x2, x3;
      ldsm_x4(kb + at((mi & 1) * 8 + (lane & 7), 2 * kk + (mi >> 1)), x0, x1, x2, x3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (kk & 1) mma16<F16>(sd[nt], x0, x1, x2, x3, qb[nt][kk][0], qb[nt][kk][1]);
        else mma16<F16>(sc[nt], x0, x1, x2, x3, qb[nt][kk][0], qb[nt][kk][1]);
      }
    }
    // which of the unit's entries the token sees (the same ones for every row)
    const int e0 = c.s.entry(c.t);
    const bool whole = e0 + kUnit <= c.s.n && (e0 >= c.s.lo || e0 + kUnit <= a.sinks);
    bool see[2] = {true, true};  // entries g and g + 8
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = e0 + g + 8 * e;
        see[e] = j < c.s.n && (j >= c.s.lo || j < a.sinks);
      }
      // values of unseen entries may hold anything, and 0 x NaN is NaN
      const int r = lane >> 1, j = e0 + r;
      if (!(j < c.s.n && (j >= c.s.lo || j < a.sinks)))
#pragma unroll
        for (int ch = (lane & 1) * (D / 16); ch < (lane & 1) * (D / 16) + D / 16; ++ch)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + at(r, ch)), "r"(0u) : "memory");
      tc::fence_proxy_async_smem();  // before the stage's next TMA write
      __syncwarp();
    }
    uint32_t pb[NT][2], pl[NT][2];
    float fac[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = see[e >> 1] ? (sc[nt][e] + sd[nt][e]) * a.scale_log2 : -INFINITY;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = fmaxf(sc[nt][r], sc[nt][2 + r]);
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float up = fmaxf(m[nt][r], x);
        fac[nt][r] = m[nt][r] == -INFINITY ? 0.f : ex2(m[nt][r] - up);
        m[nt][r] = up;
      }
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[e] = ex2(sc[nt][e] - (finite(m[nt][e & 1]) - a.offset));
#pragma unroll
      for (int r = 0; r < 2; ++r) l[nt][r] = l[nt][r] * fac[nt][r] + (pr[r] + pr[2 + r]);
      pb[nt][0] = movmatrix_t(pack16<F16>(pr[0], pr[1]));
      pb[nt][1] = movmatrix_t(pack16<F16>(pr[2], pr[3]));
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[e] -= round16<F16>(pr[e]);
      pl[nt][0] = movmatrix_t(pack16<F16>(pr[0], pr[1]));
      pl[nt][1] = movmatrix_t(pack16<F16>(pr[2], pr[3]));
    }
    if (a.accumulate) {
      float* to = a.scores + (u0 + i) * (int64_t)(kUnit * a.rows) + g;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (8 * nt + 2 * t4 + r < rows) {
            to[(8 * nt + 2 * t4 + r) * kUnit] = sc[nt][r];
            to[(8 * nt + 2 * t4 + r) * kUnit + 8] = sc[nt][2 + r];
          }
    }
#pragma unroll
    for (int kk = 0; kk < kK; ++kk) {
      uint32_t x0, x1, x2, x3;
      ldsm_x4_t(vb + at((mi >> 1) * 8 + (lane & 7), 2 * kk + (mi & 1)), x0, x1, x2, x3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float unit[4] = {0.f, 0.f, 0.f, 0.f};
        mma16<F16>(unit, x0, x1, x2, x3, pb[nt][0], pb[nt][1]);
        mma16<F16>(unit, x0, x1, x2, x3, pl[nt][0], pl[nt][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][kk][e] = o[nt][kk][e] * fac[nt][e & 1] + unit[e];
      }
    }
    __syncwarp();
    if (i + S::kStages < count) {
      issue(p, ids, stage);
      advance(p);
      ids = page_ids(p);
    }
    if (++stage == S::kStages) stage = 0, parity ^= 1;

    const bool ends = c.t + 1 == c.s.units;
    if (!WHOLE && (ends || i + 1 == count)) {  // the piece is complete
      const bool is_whole = ends && begun == 0;
      float* pp = a.part + ((int64_t)run * 2 + (begun == 0 ? 1 : 0)) * a.rows * (D + kPad);
      if (!ends && begun == 0 && lane == 0) {
        const int64_t end = u0 + i + (c.s.units - 1 - c.t);  // the head's last unit
        a.open[run] = make_int4(c.b, c.pair, run_of(end, length), 0);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sum = column_sum(l[nt][r]);
          const int row = 8 * nt + 2 * t4 + r;
          if (row >= rows) continue;
          const int j = h * a.groups + r0 + row;
          if (is_whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int64_t to = c.b * a.out_sb + j * a.out_sh;
#pragma unroll
            for (int kk = 0; kk < kK; ++kk) {
              store_out<F16>(a, to + 16 * kk + g, o[nt][kk][r] * inv);
              store_out<F16>(a, to + 16 * kk + 8 + g, o[nt][kk][2 + r] * inv);
            }
            if (g == 0) {
              const float lse2 = finite(m[nt][r]) - a.offset + log2f(sum);
              a.lse[(int64_t)c.b * a.kv * a.groups + j] = lse2 * kLn2;
              a.lse2[(int64_t)c.b * a.kv * a.groups + j] = lse2;
            }
          } else {
            float* to = pp + row * (D + kPad);
#pragma unroll
            for (int kk = 0; kk < kK; ++kk) {
              to[16 * kk + g] = o[nt][kk][r];
              to[16 * kk + 8 + g] = o[nt][kk][2 + r];
            }
            if (g == 0) to[D] = m[nt][r], to[D + 1] = sum;
          }
        }
      fresh = true;
    }
    advance(c);
  }
  if (!ok)  // loads in flight land before the CTA's shared memory is given up
    for (int64_t u = i; u < paged::ring_issued(i, S::kStages, count); ++u) {
      const paged::RingWait w = paged::ring_wait(u, S::kStages);
      tc::mbar_wait(&s_full[warp][w.stage], w.parity, 200000000ull);
    }
  if (!WHOLE) return;

  // ---- WHOLE: the warps' parts, each in its own (now free) ring, joined by the CTA into the
  // first warp's, and the CTAs' by the cluster
  float* mine = reinterpret_cast<float*>(my_ring);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float sum = column_sum(l[nt][r]);
      const int row = 8 * nt + 2 * t4 + r;
#pragma unroll
      for (int kk = 0; kk < kK; ++kk) {
        mine[row * D + 16 * kk + g] = o[nt][kk][r];
        mine[row * D + 16 * kk + 8 + g] = o[nt][kk][2 + r];
      }
      if (g == 0) s_ml[warp][row] = make_float2(m[nt][r], sum);
    }
  __syncthreads();
  float* joined = reinterpret_cast<float*>(ring);
  for (int i = tid; i < rows * D; i += kThreads) {
    float top = -INFINITY, y = 0.f;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, s_ml[w][i / D].x);
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w)
      y += reinterpret_cast<const float*>(ring + w * S::kStages * 2 * S::kTile)[i] * ex2(s_ml[w][i / D].x - finite(top));
    joined[i] = y;  // read and written by this thread only
  }
  if (tid < rows) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, s_ml[w][tid].x);
    for (int w = 0; w < S::kWarps; ++w) sum += s_ml[w][tid].y * ex2(s_ml[w][tid].x - finite(top));
    s_joined[tid] = make_float2(top, sum);
  }
  // this CTA's warps wrote the scores of its own units; its threads add their weights
  const int h = c.pair, j0 = h * a.groups;
  int first_quarter = 0, end_quarter = 0;
  Quarter quarter;
  if (a.accumulate) {
    const int parts = ctas * S::kWarps;
    first_quarter = 4 * (int)((int64_t)c.s.units * (rank * S::kWarps) / parts) + tid;
    end_quarter = 4 * (int)((int64_t)c.s.units * ((rank + 1) * S::kWarps) / parts);
    if (first_quarter < end_quarter) quarter = Quarter(a, c.b, h, c.s, first_quarter);
  }
  cluster_sync();
  for (int i = rank * kThreads + tid; i < rows * D; i += ctas * kThreads) {
    const int row = i / D, d = i % D;
    float top = -INFINITY, sum = 0.f, y = 0.f;
    for (uint32_t k = 0; k < ctas; ++k) top = fmaxf(top, remote(&s_joined[row].x, k));
    for (uint32_t k = 0; k < ctas; ++k) {
      const float f = ex2(remote(&s_joined[row].x, k) - finite(top));
      sum += remote(&s_joined[row].y, k) * f;
      y += remote(&joined[i], k) * f;
    }
    store_out<F16>(a, c.b * a.out_sb + (j0 + row) * a.out_sh + d, sum == 0.f ? 0.f : y * (1.f / sum));
  }
  if (tid < rows) {
    float top = -INFINITY, sum = 0.f;
    for (uint32_t k = 0; k < ctas; ++k) top = fmaxf(top, remote(&s_joined[tid].x, k));
    for (uint32_t k = 0; k < ctas; ++k) sum += remote(&s_joined[tid].y, k) * ex2(remote(&s_joined[tid].x, k) - finite(top));
    const float lse2 = finite(top) - a.offset + log2f(sum);
    if (rank == 0) a.lse[(int64_t)c.b * a.kv * a.groups + j0 + tid] = lse2 * kLn2;
    s_lse[tid] = lse2 == -INFINITY ? INFINITY : lse2;  // a row without weight adds 0
  }
  cluster_sync();  // no CTA leaves while another reads its part
  if (!a.accumulate) return;
  const float* scores = a.scores + (blockIdx.x / ctas) * a.whole_units * (kUnit * a.rows);
  for (int i = first_quarter; i < end_quarter; i += kThreads) {
    quarter.add(a, i, scores, 0, s_lse);
    if (i + kThreads < end_quarter) quarter = Quarter(a, c.b, h, c.s, i + kThreads);
  }
}

// Joins the heads that no run held whole: the warps of a block share a head's rows and each
// row's pieces (the first run's in its slot 1, the others' in slot 0), rescale as they go and
// meet in shared memory. Where there are fewer query heads than runs (few sequences, many pieces
// each) block i takes query head i, all warps on its one row; else (many sequences, few pieces)
// block i looks at run i and takes the key head that it begins and does not end, if any. Blocks of
// 1024 threads where the query heads are few enough to have an SM each: one long sequence of one
// key head leaves several hundred pieces a head.
template <int D, bool F16, int THREADS>
__global__ void __launch_bounds__(THREADS)
    paged_join_kernel(const AttendArgs a, int nwarps, bool by_head) {
  constexpr int kWarps = THREADS / 32;
  constexpr int kEach = 4;  // pieces in flight per warp
  __shared__ float s_o[kWarps][D];
  __shared__ float s_ml[kWarps][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  paged::launch_next();
  paged::wait_previous();
  int b, h, r0, begin, end, run, last;  // key head h, row tile from r0 on, its rows [begin, end); first and last run
  if (by_head) {
    b = blockIdx.x / (a.kv * a.groups);
    const int j = blockIdx.x % (a.kv * a.groups), g = j % a.groups;
    h = j / a.groups, r0 = g / a.rows * a.rows, begin = g - r0, end = begin + 1;
    const Span s(a, b);
    const int64_t total = a.base[a.batch] * (a.kv * a.rt);
    const int64_t u = a.base[b] * (a.kv * a.rt) + (int64_t)(h * a.rt + g / a.rows) * s.units;
    if (s.units == 0) {
      for (int d = tid; d < D; d += THREADS) store_out<F16>(a, b * a.out_sb + j * a.out_sh + d, 0.f);
      if (tid == 0) a.lse[(int64_t)b * a.kv * a.groups + j] = -INFINITY;
      return;
    }
    const int length = run_length(total, nwarps);
    run = run_of(u, length), last = run_of(u + s.units - 1, length);
    if (run == last) return;
  } else {
    run = blockIdx.x;
    const int4 open = a.open[run];
    for (b = run; b < a.batch; b += gridDim.x)  // a sequence without entries is in no run
      if (Span(a, b).units == 0)
        for (int i = tid; i < a.kv * a.groups * D; i += THREADS) {
          store_out<F16>(a, b * a.out_sb + i / D * a.out_sh + i % D, 0.f);
          if (i % D == 0) a.lse[(int64_t)b * a.kv * a.groups + i / D] = -INFINITY;
        }
    if (open.x < 0) return;
    b = open.x, h = open.y / a.rt, r0 = open.y % a.rt * a.rows, last = open.z;
    begin = 0, end = min(a.rows, a.groups - r0);
  }
  for (int row0 = begin; row0 < end; row0 += kWarps) {
    const int n = min(end - row0, kWarps), each = kWarps / n;  // rows of this turn, warps per row
    const int row = row0 + warp / each, part = warp % each;
    float acc[D / 32];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    if (row < row0 + n) {
      for (int i0 = run + part; i0 <= last; i0 += kEach * each) {
        float y[kEach][D / 32];
        float2 ml[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          const int i = min(i0 + k * each, last);
          const float* x = a.part + (((int64_t)i * 2 + (i == run ? 1 : 0)) * a.rows + row) * (D + kPad);
#pragma unroll
          for (int e = 0; e < D / 32; ++e) y[k][e] = x[32 * e + lane];
          ml[k] = *reinterpret_cast<const float2*>(x + D);
          if (i0 + k * each > last) ml[k] = make_float2(-INFINITY, 0.f);
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          if (i0 + k * each > last) break;
          const float up = fmaxf(top, ml[k].x);
          const float f = ex2(top - finite(up)), w = ex2(ml[k].x - finite(up));
          sum = sum * f + ml[k].y * w;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) acc[e] = acc[e] * f + y[k][e] * w;
          top = up;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < D / 32; ++e) s_o[warp][32 * e + lane] = acc[e];
    if (lane == 0) s_ml[warp][0] = top, s_ml[warp][1] = sum;
    __syncthreads();
    for (int i = tid; i < n * D; i += THREADS) {
      const int r = i / D, d = i % D, j = h * a.groups + r0 + row0 + r;
      top = -INFINITY;
      for (int w = r * each; w < (r + 1) * each; ++w) top = fmaxf(top, s_ml[w][0]);
      sum = 0.f;
      float y = 0.f;
      for (int w = r * each; w < (r + 1) * each; ++w) {
        const float f = ex2(s_ml[w][0] - finite(top));
        sum += s_ml[w][1] * f;
        y += s_o[w][d] * f;
      }
      store_out<F16>(a, b * a.out_sb + j * a.out_sh + d, sum == 0.f ? 0.f : y * (1.f / sum));
      if (d == 0) {
        const float lse2 = finite(top) - a.offset + log2f(sum);
        a.lse[(int64_t)b * a.kv * a.groups + j] = lse2 * kLn2;
        a.lse2[(int64_t)b * a.kv * a.groups + j] = lse2;
      }
    }
    __syncthreads();
  }
}

// Adds the weights to the mass, from the scores in the workspace: a block takes 4 kMassThreads
// entries of one (sequence, key head), a thread four of them.
__global__ void __launch_bounds__(kMassThreads, 6)
    paged_mass_kernel(const AttendArgs a) {
  __shared__ float s_lse[64];
  paged::launch_next();
  paged::wait_previous();
  const int tid = threadIdx.x, h = blockIdx.x % a.kv, b = blockIdx.x / a.kv;
  const Span s(a, b);
  int i = blockIdx.y * kMassThreads + tid;
  if (blockIdx.y * kMassThreads >= 4 * s.units) return;
  Quarter quarter;
  if (i < 4 * s.units) quarter = Quarter(a, b, h, s, i);
  const int64_t unit = a.base[b] * (a.kv * a.rt) + (int64_t)h * a.rt * s.units;
  if (tid < a.groups) {
    const float x = a.lse2[((int64_t)b * a.kv + h) * a.groups + tid];
    s_lse[tid] = x == -INFINITY ? INFINITY : x;
  }
  __syncthreads();
  while (i < 4 * s.units) {
    quarter.add(a, i, a.scores + unit * (kUnit * a.rows), (int64_t)s.units * (kUnit * a.rows), s_lse);
    if ((i += gridDim.y * kMassThreads) < 4 * s.units) quarter = Quarter(a, b, h, s, i);
  }
}

constexpr size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// What a launch needs beside the caller's arguments: row tiles, grid, workspace layout.
struct Plan {
  int groups, rt, rows, nt, ctas, runs, cluster;
  int64_t units_per_head;
  size_t base, open, part, lse2, scores, bytes;
};

// Clusters of `size` CTAs of this kernel that the current device holds at once (one CTA fills an
// SM, and the GPCs have different numbers of them), looked up once per device and size.
int clusters_at_once(int log_size) {
  static std::atomic<int> cached[64][4] = {};
  const int size = 1 << log_size, fallback = paged_sm_count() / size - paged_sm_count() / 8 / size;
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fallback;
  if ((n = cached[dev][log_size].load(std::memory_order_relaxed)) > 0) return n;
  static std::atomic<uint64_t> done{0};
  const void* kernel = (const void*)paged_attend_kernel<128, 1, false, true>;
  if (paged_allow_smem(kernel, kRing + 1024, done) != cudaSuccess) return fallback;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)size), cfg.blockDim = dim3(32 * Shape<128>::kWarps), cfg.dynamicSmemBytes = kRing + 1024;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)size, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return fallback;
  }
  cached[dev][log_size].store(n, std::memory_order_relaxed);
  return n;
}

// log2 of the CTAs per key head where a cluster takes a whole head (one launch, no workspace
// without weights), -1 where the equal runs and their join are better. The join costs about 6 us at
// any size; a cluster costs the SMs that its size leaves over and, with ragged lengths, the time
// of the longest sequence. So it is for heads whose clusters the device holds at once and CTAs
// that walk at most kClusterUnits units, by the table's capacity (128 heads of 4000 entries, runs
// and clusters: 51 and 45 us; 96 heads: 42 and 36 us; with lengths spread over 1 .. 4000: 33 and
// 34, 30 and 33 us). The cluster is the largest that leaves every warp two units. A CTA alone reads
// some 75 GB/s, so that clusters on few of the SMs fall behind earlier (16 heads of 16000 entries on
// 64 CTAs: 34 us; the runs take 21 us for lengths spread over 1 .. 16000). Heads of
// several row tiles take the runs: two clusters would add to the same mass, and asking for the
// weights is not to change a result's bits.
int head_cluster(int64_t heads, int64_t units_per_head, int row_tiles) {
  if (row_tiles > 1 || heads > paged_sm_count()) return -1;
  int c = 0;
  while (c < 3 && units_per_head > (int64_t)2 * Shape<128>::kWarps << c && heads <= clusters_at_once(c + 1)) ++c;
  const int most = 5 * (heads << c) >= 3 * paged_sm_count() ? kClusterUnits : kClusterUnits / 2;
  return units_per_head <= (int64_t)most << c ? c : -1;
}

Plan make_plan(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_attend_desc& d) {
  Plan p;
  p.groups = d.h / c.kv;
  p.rt = (p.groups + 15) / 16;
  p.rows = (p.groups + p.rt - 1) / p.rt;
  p.nt = p.rows <= 8 ? 1 : 2;
  const int warps = c.d == 256 ? Shape<256>::kWarps : Shape<128>::kWarps;
  // the most units that the table allows
  const int64_t cap = (int64_t)b.width * c.page;
  int64_t per = (cap + kUnit - 1) / kUnit;
  if (d.window > 0) {
    const int64_t bound = ((int64_t)d.sinks + kUnit - 1) / kUnit + ((int64_t)d.window + kUnit - 1) / kUnit + 1;
    if (bound < per) per = bound;
  }
  p.units_per_head = per;
  const int64_t heads = (int64_t)b.batch * c.kv, units = per * heads * p.rt;
  const int sms = paged_sm_count();
  const int log_cluster = head_cluster(heads, per, p.rt);
  p.cluster = log_cluster < 0 ? 0 : 1 << log_cluster;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  p.base = p.open = p.part = p.lse2 = p.scores = 0;
  if (p.cluster > 0) {
    p.ctas = (int)heads * p.cluster, p.runs = 0;
  } else {
    // short work is spread over all SMs, one warp each, before a second warp of an SM gets any
    const int64_t spread = (units + kMinUnits - 1) / kMinUnits;
    p.ctas = (int)(spread < 1 ? 1 : spread < sms ? spread : sms);
    p.runs = p.ctas * warps;
    p.base = take(((size_t)b.batch + 1) * 8);
    p.open = take((size_t)p.runs * 16);
    p.part = take((size_t)p.runs * 2 * p.rows * (c.d + kPad) * 4);
    p.lse2 = take((size_t)b.batch * d.h * 4);
  }
  if (d.accumulate) p.scores = take((size_t)units * kUnit * p.rows * 4);
  p.bytes = at;
  return p;
}

template <int D, int NT, bool F16, bool WHOLE>
cudaError_t launch_kernel(const AttendArgs& a, const Plan& p, const CUtensorMap& mk, const CUtensorMap& mv,
                          cudaStream_t st) {
  constexpr int smem = kRing + 1024;
  static std::atomic<uint64_t> done{0};
  auto* kernel = paged_attend_kernel<D, NT, F16, WHOLE>;
  const cudaError_t e = paged_allow_smem((const void*)kernel, smem, done);
  if (e != cudaSuccess) return e;
  return launch_after(kernel, dim3((unsigned)p.ctas), dim3(32 * Shape<D>::kWarps), smem, st, WHOLE ? p.cluster : 1, mk, mv, a);
}

template <int D, int NT, bool F16>
cudaError_t launch(const AttendArgs& a, const Plan& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  if (p.cluster > 0) return launch_kernel<D, NT, F16, true>(a, p, mk, mv, st);
  const cudaError_t e = launch_kernel<D, NT, F16, false>(a, p, mk, mv, st);
  if (e != cudaSuccess) return e;
  const int64_t query_heads = (int64_t)a.batch * a.kv * a.groups;
  const bool by_head = query_heads <= p.runs;
  const dim3 grid((unsigned)(by_head ? query_heads : p.runs));
  const cudaError_t j = by_head && query_heads <= paged_sm_count()
                            ? launch_after(paged_join_kernel<D, F16, 1024>, grid, dim3(1024), 0, st, 1, a, p.runs, by_head)
                            : launch_after(paged_join_kernel<D, F16, 256>, grid, dim3(256), 0, st, 1, a, p.runs, by_head);
  if (j != cudaSuccess || !a.accumulate || p.units_per_head == 0) return j;
  const int64_t slices = (p.units_per_head * 4 + kMassThreads - 1) / kMassThreads;
  return launch_after(paged_mass_kernel,
                      dim3((unsigned)((int64_t)a.batch * a.kv), (unsigned)(slices < 65535 ? slices : 65535)),
                      dim3(kMassThreads), 0, st, 1, a);
}

template <int D>
cudaError_t launch_d(const AttendArgs& a, const Plan& p, bool f16, const CUtensorMap& mk, const CUtensorMap& mv,
                     cudaStream_t st) {
  if (p.nt == 1) return f16 ? launch<D, 1, true>(a, p, mk, mv, st) : launch<D, 1, false>(a, p, mk, mv, st);
  return f16 ? launch<D, 2, true>(a, p, mk, mv, st) : launch<D, 2, false>(a, p, mk, mv, st);
}

}  // namespace

size_t paged_attend_workspace(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_attend_desc& d) {
  return make_plan(c, b, d).bytes;
}

cudaError_t launch_paged_attend(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_attend_desc& d,
                                void* ws, cudaStream_t st) {
  const Plan p = make_plan(c, b, d);
  AttendArgs a = {};
  a.table = b.block_table, a.table_stride = b.table_stride, a.lengths = b.lengths;
  a.batch = b.batch, a.width = c.pages > 0 ? b.width : 0, a.page = c.page, a.log_page = paged_log2(c.page);
  a.kv = c.kv, a.groups = p.groups, a.rt = p.rt, a.rows = p.rows;
  a.window = d.window, a.sinks = d.sinks, a.accumulate = d.accumulate;
  a.scale_log2 = d.scale * 1.4426950408889634f;
  a.offset = c.dtype == PBK_F16 ? 14.f : 0.f;
  a.q = static_cast<const uint16_t*>(d.q), a.q_sb = d.q_stride_b, a.q_sh = d.q_stride_h;
  a.out = d.out, a.out_sb = d.out_stride_b, a.out_sh = d.out_stride_h, a.out_f32 = d.out_dtype == PBK_F32;
  a.lse = d.lse;
  a.mass = c.mass, a.meta_page = c.meta_page, a.meta_head = c.meta_head, a.pages = c.pages;
  uint8_t* w = static_cast<uint8_t*>(ws);
  a.base = reinterpret_cast<int64_t*>(w + p.base);
  a.open = reinterpret_cast<int4*>(w + p.open);
  a.part = reinterpret_cast<float*>(w + p.part);
  a.lse2 = reinterpret_cast<float*>(w + p.lse2);
  a.scores = reinterpret_cast<float*>(w + p.scores);
  a.whole_units = p.units_per_head;
  a.err = device_error_word();
  CUtensorMap mk, mv;
  {
    // [64 elements][entries of a page][64-element blocks of the head][heads][pages]
    const bool any = c.pages > 0;  // no pages: nothing is read, and the strides may be anything
    const uint64_t dims[5] = {64, (uint64_t)c.page, (uint64_t)(c.d / 64), (uint64_t)c.kv, any ? (uint64_t)c.pages : 1};
    const uint64_t strides[4] = {any ? (uint64_t)c.stride_entry * 2 : 512, 128, any ? (uint64_t)c.stride_head * 2 : 512,
                                 any ? (uint64_t)c.stride_page * 2 : 512};
    const uint32_t box[5] = {64, (uint32_t)(c.page < kUnit ? c.page : kUnit), (uint32_t)(c.d / 64), 1, 1};
    const void* k = any ? c.k_pages : d.q;
    const void* v = any ? c.v_pages : d.q;
    if (!make_tmap_bf16_sw128(&mk, k, 5, dims, strides, box) || !make_tmap_bf16_sw128(&mv, v, 5, dims, strides, box))
      return cudaErrorInvalidValue;
  }
  const bool f16 = c.dtype == PBK_F16;
  if (c.d == 64) return launch_d<64>(a, p, f16, mk, mv, st);
  if (c.d == 128) return launch_d<128>(a, p, f16, mk, mv, st);
  return launch_d<256>(a, p, f16, mk, mv, st);
}

}  // namespace pbk
