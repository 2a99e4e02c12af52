// Attention of one new token per sequence over the paged cache.
//
// The work is cut into units of 16 entries of one (sequence, key head, row tile): a row tile is
// up to 16 of the query heads that share the key head. All units of a launch stand in one line
// (sequence by sequence, head by head, entry by entry) and every warp of the grid takes an equal
// run of it, so ragged lengths, one long sequence and many short ones load the SMs alike. A warp
// walks its run with an online softmax (base 2) and writes a head's result when its run holds
// the whole head, else the partial (maximum, sum, weighted values) of its piece; the join
// kernel, launched behind it, merges the pieces of each head and, when asked, turns the scores
// kept in the workspace into weights and adds them to the cache's mass.
#include "common.cuh"
#include "paged.cuh"
#include "tc.cuh"
#include "tma_host.h"

namespace pbk {
namespace {

constexpr int kUnit = 16;           // entries per unit
constexpr int kRing = 192 * 1024;   // staging bytes per CTA
constexpr int kMinUnits = 2;        // units per warp below which fewer warps take part
constexpr int kJoinThreads = 256;
constexpr int kSlice = 2048;        // entries per CTA of the mass update

template <int D>
struct Shape {
  static constexpr int kWarps = D == 256 ? 4 : 8;
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
  float* part;               // [warps][2][rows][D + 2]
  float* lse2;               // [batch, h] base 2, of the heads that one warp held whole
  float* scores;             // [units][16][score_stride] base 2
  int score_stride, d;
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
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w, int v) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(tc::smem_u32(dst)),
      "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v)
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

__device__ __forceinline__ int64_t run_start(int64_t total, int warps, int w) { return total * w / warps; }
// The warp whose run holds unit u.
__device__ __forceinline__ int run_of(int64_t total, int warps, int64_t u) {
  return (int)(((u + 1) * warps - 1) / total);
}
__device__ __forceinline__ int active_warps(int64_t total, int warps) {
  const int64_t w = (total + kMinUnits - 1) / kMinUnits;
  return w < warps ? (w > 0 ? (int)w : 1) : warps;
}

__device__ __forceinline__ void store_out(const AttendArgs& a, bool f16, int64_t at, float y) {
  if (a.out_f32) static_cast<float*>(a.out)[at] = y;
  else if (f16) static_cast<__half*>(a.out)[at] = __float2half_rn(y);
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
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
// Weights enter the product with V as 16-bit numbers: fp16 as one (11 bits), bf16 as two (the
// rounded weight and what the rounding left, 16 bits together), so that the result's own
// rounding is the largest error; the second product runs in the tensor cores' idle time.
template <int D, int NT, bool F16>
__global__ void __launch_bounds__(32 * Shape<D>::kWarps, 1)
    paged_attend_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                        const AttendArgs a) {
  using S = Shape<D>;
  constexpr int kK = D / 16;
  constexpr int kThreads = 32 * S::kWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t s_full[S::kWarps][S::kStages];
  __shared__ int64_t s_sum[S::kWarps];
  __shared__ int64_t s_off[S::kWarps];
  __shared__ int s_seq[S::kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nwarps = gridDim.x * S::kWarps;
  const int pairs = a.kv * a.rt;  // (key head, row tile) of a sequence
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

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
  if (lane < S::kStages) tc::mbar_init(&s_full[warp][lane], 1);
  if (lane == 0) {
    s_seq[warp] = -1;
    tc::fence_barrier_init();
  }
  __syncthreads();
  int64_t total = 0;
  before -= mine;
#pragma unroll
  for (int w = 0; w < S::kWarps; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  if (blockIdx.x == 0) {
    int64_t at = before;
    for (int b = b0; b < b1; ++b) {
      a.base[b] = at;
      at += Span(a, b).units;
    }
    if (tid == 0) a.base[a.batch] = total;
  }
  total *= pairs;
  const int active = active_warps(total, nwarps);
  if (total > 0) {
    int64_t at = before;
    for (int b = b0; b < b1; ++b) {
      const int64_t len = Span(a, b).units;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const int run = w * gridDim.x + blockIdx.x;  // neighbouring runs on different SMs
        if (run < active) {
          const int64_t u = run_start(total, active, run);
          if (u >= at * pairs && u < (at + len) * pairs) s_seq[w] = b, s_off[w] = u - at * pairs;
        }
      }
      at += len;
    }
  }
  __syncthreads();
  if (s_seq[warp] < 0) return;
  const int run = warp * gridDim.x + blockIdx.x;
  const int64_t u0 = run_start(total, active, run);
  const int count = (int)(run_start(total, active, run + 1) - u0);

  // ---- producer and consumer positions in the line of units
  struct Walk {
    int b, pair, t;
    Span s;
  };
  Walk c;
  c.b = s_seq[warp];
  c.s = Span(a, c.b);
  c.pair = (int)(s_off[warp] / c.s.units);
  c.t = (int)(s_off[warp] % c.s.units);
  Walk p = c;
  auto advance = [&](Walk& w) {
    if (++w.t < w.s.units) return;
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
    if (w.b >= a.batch) return make_int2(-1, -1);
    const int32_t* row = a.table + w.b * a.table_stride;
    const int i = w.s.entry(w.t) >> a.log_page;
    return make_int2(row[i], small && i + 1 < a.width ? row[i + 1] : -1);
  };
  uint8_t* my_ring = ring + warp * S::kStages * 2 * S::kTile;
  auto issue = [&](const Walk& w, int2 ids, int stage) {
    if (lane == 0) {
      uint64_t* bar = &s_full[warp][stage];
      uint8_t* k = my_ring + stage * 2 * S::kTile;
      uint8_t* v = k + S::kTile;
      const int h = w.pair / a.rt, row = w.s.entry(w.t) & (a.page - 1);
      tc::mbar_expect_tx(bar, 2 * S::kTile);
      tma_load_5d(k, &mk, bar, 0, row, 0, h, ids.x);
      tma_load_5d(v, &mv, bar, 0, row, 0, h, ids.x);
      if (small) {
        tma_load_5d(k + S::kTile / 2, &mk, bar, 0, 0, 0, h, ids.y);
        tma_load_5d(v + S::kTile / 2, &mv, bar, 0, 0, 0, h, ids.y);
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
  int rows = 0;
  bool fresh = true, ok = true;
  int begun = c.t;  // first unit of the current piece in its head
  int stage = 0;
  uint32_t parity = 0;

  for (int i = 0; i < count; ++i) {
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
    bool raised = false;
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
        raised |= up != m[nt][r];
        m[nt][r] = up;
      }
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[e] = ex2(sc[nt][e] - (finite(m[nt][e & 1]) - a.offset));
#pragma unroll
      for (int r = 0; r < 2; ++r) l[nt][r] = l[nt][r] * fac[nt][r] + (pr[r] + pr[2 + r]);
      pb[nt][0] = movmatrix_t(pack16<F16>(pr[0], pr[1]));
      pb[nt][1] = movmatrix_t(pack16<F16>(pr[2], pr[3]));
      if (!F16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] -= __bfloat162float(__float2bfloat16_rn(pr[e]));
        pl[nt][0] = movmatrix_t(pack16<F16>(pr[0], pr[1]));
        pl[nt][1] = movmatrix_t(pack16<F16>(pr[2], pr[3]));
      }
    }
    if (a.accumulate) {
      float* to = a.scores + (u0 + i) * (int64_t)(kUnit * a.score_stride);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (8 * nt + 2 * t4 < a.score_stride) {
          *reinterpret_cast<float2*>(to + g * a.score_stride + 8 * nt + 2 * t4) = make_float2(sc[nt][0], sc[nt][1]);
          *reinterpret_cast<float2*>(to + (g + 8) * a.score_stride + 8 * nt + 2 * t4) = make_float2(sc[nt][2], sc[nt][3]);
        }
    }
    if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int kk = 0; kk < kK; ++kk) {
          o[nt][kk][0] *= fac[nt][0];
          o[nt][kk][1] *= fac[nt][1];
          o[nt][kk][2] *= fac[nt][0];
          o[nt][kk][3] *= fac[nt][1];
        }
    }
#pragma unroll
    for (int kk = 0; kk < kK; ++kk) {
      uint32_t x0, x1, x2, x3;
      ldsm_x4_t(vb + at((mi >> 1) * 8 + (lane & 7), 2 * kk + (mi & 1)), x0, x1, x2, x3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma16<F16>(o[nt][kk], x0, x1, x2, x3, pb[nt][0], pb[nt][1]);
        if (!F16) mma16<F16>(o[nt][kk], x0, x1, x2, x3, pl[nt][0], pl[nt][1]);
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
    if (ends || i + 1 == count) {  // the piece is complete
      const bool is_whole = ends && begun == 0;
      float* pp = a.part + ((int64_t)run * 2 + (begun == 0 ? 1 : 0)) * a.rows * (D + 2);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float sum = l[nt][r];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int row = 8 * nt + 2 * t4 + r;
          if (row >= rows) continue;
          const int j = h * a.groups + r0 + row;
          if (is_whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int64_t to = c.b * a.out_sb + j * a.out_sh;
#pragma unroll
            for (int kk = 0; kk < kK; ++kk) {
              store_out(a, F16, to + 16 * kk + g, o[nt][kk][r] * inv);
              store_out(a, F16, to + 16 * kk + 8 + g, o[nt][kk][2 + r] * inv);
            }
            if (g == 0) {
              const float lse2 = finite(m[nt][r]) - a.offset + log2f(sum);
              a.lse[(int64_t)c.b * a.kv * a.groups + j] = lse2 * 0.6931471805599453f;
              a.lse2[(int64_t)c.b * a.kv * a.groups + j] = lse2;
            }
          } else {
            float* to = pp + row * (D + 2);
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
    for (int s = 0; s < S::kStages; ++s) tc::mbar_wait(&s_full[warp][s], parity, 200000000ull);
}

// The pieces of one (sequence, key head, row tile): runs first .. last, the first one's in its
// slot 1, the others' in slot 0.
struct Pieces {
  int first, last;
  __device__ Pieces(const AttendArgs& a, int64_t base, int units, int pair, int64_t total, int active) {
    const int64_t u = base * (a.kv * a.rt) + (int64_t)pair * units;
    first = run_of(total, active, u);
    last = run_of(total, active, u + units - 1);
  }
  __device__ const float* at(const AttendArgs& a, int run, int row) const {
    return a.part + (((int64_t)run * 2 + (run == first ? 1 : 0)) * a.rows + row) * (a.d + 2);
  }
};

// (maximum, sum of exponentials) over the pieces, the same in every lane of the warp.
__device__ __forceinline__ float2 join_row(const AttendArgs& a, const Pieces& pc, int row, int lane) {
  float top = -INFINITY;
  for (int i = pc.first + lane; i <= pc.last; i += 32) top = fmaxf(top, pc.at(a, i, row)[a.d]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.f;
  for (int i = pc.first + lane; i <= pc.last; i += 32) {
    const float* x = pc.at(a, i, row) + a.d;
    sum += x[1] * ex2(x[0] - finite(top));
  }
  return make_float2(top, warp_sum(sum));
}

// Blocks below batch * h join the pieces of one query head; the others add the weights of kSlice
// entries of one (sequence, key head) to the mass, from the scores in the workspace.
template <int D, bool F16>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_kernel(const AttendArgs a, int nwarps, int slices) {
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float s_o[kWarps][D];
  __shared__ float s_lse[64];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = a.kv * a.groups;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t total = a.base[a.batch] * (a.kv * a.rt);
  const int active = active_warps(total, nwarps);
  int64_t id = blockIdx.x;
  if (id < (int64_t)a.batch * heads) {
    const int b = (int)(id / heads), j = (int)(id % heads);
    const Span s(a, b);
    const int64_t to = b * a.out_sb + j * a.out_sh;
    if (s.units == 0) {
      for (int d = tid; d < D; d += kJoinThreads) store_out(a, F16, to + d, 0.f);
      if (tid == 0) a.lse[id] = -INFINITY;
      return;
    }
    const int h = j / a.groups, r = j % a.groups, pair = h * a.rt + r / a.rows, row = r % a.rows;
    const Pieces pc(a, a.base[b], s.units, pair, total, active);
    if (pc.first == pc.last) return;  // one warp held it whole
    const float2 ms = join_row(a, pc, row, lane);
    const float inv = ms.y == 0.f ? 0.f : 1.f / ms.y;
    float acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
    for (int i = pc.first + warp; i <= pc.last; i += kWarps) {
      const float* x = pc.at(a, i, row);
      const float f = ex2(x[D] - finite(ms.x));
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] += f * x[32 * e + lane];
    }
#pragma unroll
    for (int e = 0; e < D / 32; ++e) s_o[warp][32 * e + lane] = acc[e];
    __syncthreads();
    for (int d = tid; d < D; d += kJoinThreads) {
      float y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) y += s_o[w][d];
      store_out(a, F16, to + d, y * inv);
    }
    if (tid == 0) a.lse[id] = (finite(ms.x) - a.offset + log2f(ms.y)) * 0.6931471805599453f;
    return;
  }
  id -= (int64_t)a.batch * heads;
  const int slice = (int)(id % slices), h = (int)(id / slices % a.kv), b = (int)(id / slices / a.kv);
  const Span s(a, b);
  const int t0 = slice * (kSlice / kUnit), t1 = min(t0 + kSlice / kUnit, s.units);
  if (t0 >= t1) return;
  const int64_t base = a.base[b];
  for (int r = warp; r < a.groups; r += kWarps) {
    const Pieces pc(a, base, s.units, h * a.rt + r / a.rows, total, active);
    float lse2;
    if (pc.first == pc.last) {
      lse2 = a.lse2[(int64_t)b * heads + h * a.groups + r];
    } else {
      const float2 ms = join_row(a, pc, r % a.rows, lane);
      lse2 = finite(ms.x) - a.offset + log2f(ms.y);
    }
    if (lane == 0) s_lse[r] = lse2;
  }
  __syncthreads();
  for (int i = tid; i < (t1 - t0) * kUnit; i += kJoinThreads) {
    const int t = t0 + i / kUnit, e = s.entry(t) + i % kUnit;
    if (e >= s.n) continue;
    const int page = paged::page_of(a.table + b * a.table_stride, e, a.log_page, a.pages);
    if (page < 0) continue;
    float sum = 0.f;
    for (int rt = 0; rt < a.rt; ++rt) {
      const int64_t u = base * (a.kv * a.rt) + (int64_t)(h * a.rt + rt) * s.units + t;
      const float* x = a.scores + (u * kUnit + i % kUnit) * a.score_stride;
      const int rows = min(a.rows, a.groups - rt * a.rows);
      for (int r = 0; r < rows; ++r) {
        const float lse2 = s_lse[rt * a.rows + r];
        sum += lse2 == -INFINITY ? 0.f : ex2(x[r] - lse2);
      }
    }
    a.mass[page * a.meta_page + h * a.meta_head + (e & (a.page - 1))] += sum;
  }
}

constexpr size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// What a launch needs beside the caller's arguments: row tiles, grid, workspace layout.
struct Plan {
  int groups, rt, rows, nt, warps_per_cta, ctas, score_stride, slices;
  size_t base, part, lse2, scores, bytes;
};

int sm_count() {
  static int cached[64] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) cached[dev] = n;
  return cached[dev] > 0 ? cached[dev] : 148;
}

Plan make_plan(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_attend_desc& d) {
  Plan p;
  p.groups = d.h / c.kv;
  p.rt = (p.groups + 15) / 16;
  p.rows = (p.groups + p.rt - 1) / p.rt;
  p.nt = p.rows <= 8 ? 1 : 2;
  p.warps_per_cta = c.d == 256 ? 4 : 8;
  // the most units that the table allows
  const int64_t cap = (int64_t)b.width * c.page;
  int64_t per = (cap + kUnit - 1) / kUnit;
  if (d.window > 0) {
    const int64_t bound = ((int64_t)d.sinks + kUnit - 1) / kUnit + ((int64_t)d.window + kUnit - 1) / kUnit + 1;
    if (bound < per) per = bound;
  }
  const int64_t units = per * b.batch * c.kv * p.rt;
  const int sms = sm_count();
  // short work is spread over all SMs, one warp each, before a second warp of an SM gets any
  const int64_t spread = (units + kMinUnits - 1) / kMinUnits;
  p.ctas = (int)(spread < 1 ? 1 : spread < sms ? spread : sms);
  p.score_stride = (p.rows + 1) / 2 * 2;
  p.slices = (int)((per * kUnit + kSlice - 1) / kSlice);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  p.base = take(((size_t)b.batch + 1) * 8);
  p.part = take((size_t)p.ctas * p.warps_per_cta * 2 * p.rows * (c.d + 2) * 4);
  p.lse2 = take((size_t)b.batch * d.h * 4);
  p.scores = d.accumulate ? take((size_t)units * kUnit * p.score_stride * 4) : 0;
  p.bytes = at;
  return p;
}

template <int D, int NT, bool F16>
cudaError_t launch(const AttendArgs& a, const Plan& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  using S = Shape<D>;
  constexpr int smem = kRing + 1024;
  auto* kernel = paged_attend_kernel<D, NT, F16>;
  cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<p.ctas, 32 * S::kWarps, smem, st>>>(mk, mv, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  const int64_t blocks = (int64_t)a.batch * a.kv * a.groups + (a.accumulate ? (int64_t)a.batch * a.kv * p.slices : 0);
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, F16>, a, p.ctas * S::kWarps, p.slices);
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
  a.part = reinterpret_cast<float*>(w + p.part);
  a.lse2 = reinterpret_cast<float*>(w + p.lse2);
  a.scores = reinterpret_cast<float*>(w + p.scores);
  a.score_stride = p.score_stride, a.d = c.d;
  a.err = device_error_word();
  CUtensorMap mk, mv;
  {
    // [64 elements][entries of a page][64-element blocks of the head][heads][pages]
    const bool any = c.pages > 0;  // no pages: nothing is read, and the strides may be anything
    const uint64_t dims[5] = {64, (uint64_t)c.page, (uint64_t)(c.d / 64), (uint64_t)c.kv, any ? (uint64_t)c.pages : 1};
    const uint64_t strides[4] = {any ? (uint64_t)c.stride_entry * 2 : 512, 128, any ? (uint64_t)c.stride_head * 2 : 512,
                                 any ? (uint64_t)c.stride_page * 2 : 512};
    const uint32_t box[5] = {64, (uint32_t)(c.page < kUnit ? c.page : kUnit), (uint32_t)(c.d / 64), 1, 1};
    const void* k = any ? c.k_pages : ws;
    const void* v = any ? c.v_pages : ws;
    if (!make_tmap_bf16_sw128(&mk, k, 5, dims, strides, box) || !make_tmap_bf16_sw128(&mv, v, 5, dims, strides, box))
      return cudaErrorInvalidValue;
  }
  const bool f16 = c.dtype == PBK_F16;
  if (c.d == 64) return launch_d<64>(a, p, f16, mk, mv, st);
  if (c.d == 128) return launch_d<128>(a, p, f16, mk, mv, st);
  return launch_d<256>(a, p, f16, mk, mv, st);
}

}  // namespace pbk
