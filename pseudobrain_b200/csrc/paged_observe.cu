// The attention weights of a prompt's last queries over the paged cache, summed into its mass.
//
// For every (sequence, key head) there are rows = queries x query heads of the key head, and
// mass_j += sum_r 2^(s_rj - lse_r) with s = c q.k (c = scale log2 e) over the entries j that row r
// sees. The rows' logarithms come first, so the scores are computed twice:
//   pass 1: S = Q K^T   (tcgen05, M = 128 rows, N = 128 entries): a thread holds one row of the
//           tile and keeps its running maximum and sum, no exchange between threads;
//   pass 2: S^T = K Q^T (M = 128 entries, N = rows): a thread holds one entry and sums its
//           weights over the rows, then adds them to the mass once. No atomics.
// Storing the scores instead would cost 4 bytes per (row, entry), more than the keys themselves
// from 64 rows of a head of 128 on.
//
// Keys are cut into tiles of 128 entries of one (sequence, key head); all tiles stand in one line
// and each CTA (one per SM) takes an equal run of it. Row tiles hold as many whole queries as fit
// 128 rows; up to kMaxTiles of them share each key tile, more take further launches. Warps: 0 and
// 18 TMA producers (a key tile is up to 64 boxes, page by page, and one warp issues a box in
// about 45 ns; queries come as one box of heads x queries), 1 MMA issuer, 2-17 four groups that
// take the key tiles in turn, each from its own accumulator in TMEM (pass 2 over 131072 entries
// and 8 heads: 66 us with two groups, 60 with four). Every wait is bounded; on timeout the kernel
// records an error code and winds down.
//
// What bounds it: per key tile and pass 128 x 128 exponentials (16 a clock and SM: 0.55 us), the
// keys' bytes (32 KB at an SM's share of HBM: 0.75 us) and 0.37 us of MMA.
#include <atomic>

#include "common.cuh"
#include "paged.cuh"
#include "tc.cuh"
#include "tma_host.h"

namespace pbk {
namespace {

constexpr int kTile = 128;       // entries of a key tile, rows of a row tile
constexpr int kMaxTiles = 8;     // row tiles of a launch
constexpr int kProducers = 2;    // producer warps: warp 0 and the one after the epilogue's
constexpr int kGroups = 4;       // epilogue groups of four warps, each with an accumulator in TMEM
constexpr int kEpilogue = 128 * kGroups;
constexpr int kThreads = 32 * (kProducers + 1) + kEpilogue;
constexpr uint32_t kTmemCols = 512;

// Stages of the key and query rings. One row tile (ONE) stays for all of a head's key tiles, and
// the keys get what is left: a saturated HBM takes some 4 us to answer, which 192 KB in flight
// per SM just cover. More row tiles pass by once per key tile, out of L2.
template <int D, bool ONE>
struct Shape {
  static constexpr int kBytes = kTile * D * 2;  // a tile of keys or queries
  static constexpr int kBlock = kTile * 128;    // its 64-element columns: 128 rows of 128 bytes
  static constexpr int kKeys = ONE ? (D == 64 ? 12 : D == 128 ? 6 : 2) : (D == 64 ? 5 : D == 128 ? 3 : 1);
  static constexpr int kQueries = ONE ? 1 : D == 64 ? 5 : D == 128 ? 3 : 2;
  static constexpr int kSmem = (kKeys + kQueries) * kBytes + 1024;
};

struct ObserveArgs {
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  int batch, width, page, log_page, pages;
  int kv, groups, queries;       // key heads, query heads per key head, queries of the whole call
  int w0, nw, tiles;             // first query of this launch, queries per row tile, row tiles
  float c;                       // scale log2 e
  float* mass;
  int64_t meta_page, meta_head;
  float2* part;                  // [CTAs][2][tiles * 128] (maximum, sum) of a run's unfinished heads
  float* lse;                    // [batch][kv][tiles * 128] base 2, of heads that one run held whole
  int* err;
};

// A maximum over no scores (or over -inf alone) as 0: 2^(-inf - 0) is then 0 without a branch.
__device__ __forceinline__ float finite(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 operations in one instruction (fma.rn.f32x2 and add.rn.f32x2 round each half like the
// scalar ones).
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// sum[i & 3] += 2^(x c + d) over 16 scores, in three rounds of independent instructions.
__device__ __forceinline__ void add_exps(uint64_t (&sum)[4], const uint32_t* x, uint64_t c, const uint64_t (&d)[8]) {
  uint64_t y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fma2(pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), c, d[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 z = unpack2(y[i]);
    y[i] = pack2(ex2(z.x), ex2(z.y));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i & 3] = add2(sum[i & 3], y[i]);
}
// L2 cache policies: leave first, stay.
__device__ __forceinline__ uint64_t policy_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t policy_last() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
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
// Waits for this thread's TMEM loads and ties the registers to the wait.
__device__ __forceinline__ void landed(uint32_t (&x)[32]) {
  tc::tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(x[i]));
}
__device__ __forceinline__ void group_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kEpilogue) : "memory"); }

// A CTA's run of the line of key tiles, one head at a time.
struct Run {
  int b, h, t, n, tiles, count;  // the head, its tiles t .. t + count - 1 of the run; the sequence's length and tiles
  int64_t left;                  // tiles of the run from this head on, its own among them
  __device__ void load(const ObserveArgs& a) {
    n = paged::clamp_length(a.lengths[b], a.width, a.page);
    tiles = (n + kTile - 1) / kTile;
  }
  __device__ void start(const ObserveArgs& a, int b_, int64_t at, int64_t length) {  // at: its first tile in sequence b_
    b = b_, left = length, h = t = count = 0;
    load(a);
    if (left == 0) return;
    h = (int)(at / tiles), t = (int)(at % tiles);
    count = (int)min(left, (int64_t)(tiles - t));
  }
  __device__ void next(const ObserveArgs& a) {
    left -= count;
    if (left == 0) return;
    if (++h == a.kv) {
      h = 0;
      do {
        ++b;
        load(a);
      } while (tiles == 0);
    }
    t = 0, count = (int)min(left, (int64_t)tiles);
  }
};

template <int D, bool F16, bool ONE, int PASS>
__global__ void __launch_bounds__(kThreads, 1)
    paged_observe_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                         const ObserveArgs a) {
  using S = Shape<D, ONE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* keys = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* queries = keys + S::kKeys * S::kBytes;
  __shared__ uint64_t k_full[S::kKeys], k_empty[S::kKeys], q_full[S::kQueries], q_empty[S::kQueries], s_full[kGroups],
      s_empty[kGroups], drain;
  constexpr int kRows = ONE ? kTile : kMaxTiles * kTile;
  // pass 1: the groups' (maximum, sum) per row; of one row tile joined at the end, group by group
  __shared__ float2 s_stat[PASS == 1 && !ONE ? kGroups : 1][PASS == 1 ? kRows : 1];
  __shared__ __align__(16) float s_lse[PASS == 2 ? kRows : 4];  // pass 2: negated
  __shared__ int s_place[PASS == 2 ? kRows : 1];
  __shared__ int64_t s_sum[kThreads / 32], s_off;
  __shared__ int s_seq;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  paged::launch_next();

  if (tid == 0) {
    for (int s = 0; s < S::kKeys; ++s) tc::mbar_init(&k_full[s], 1), tc::mbar_init(&k_empty[s], 1);
    for (int s = 0; s < S::kQueries; ++s) tc::mbar_init(&q_full[s], 1), tc::mbar_init(&q_empty[s], 1);
    for (int s = 0; s < kGroups; ++s) tc::mbar_init(&s_full[s], 1), tc::mbar_init(&s_empty[s], 128);
    tc::mbar_init(&drain, 1);
    abort_flag = 0;
    s_seq = -1;
    tc::fence_barrier_init();
    tc::prefetch_tmap(&mq);
    tc::prefetch_tmap(&mk);
  }
  if (warp == 1) {
    tc::tmem_alloc(&tmem_base, kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  paged::wait_previous();

  // ---- this CTA's run: a scan of the sequences' tiles
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  auto tiles_of = [&](int b) {
    return (paged::clamp_length(a.lengths[b], a.width, a.page) + kTile - 1) / kTile;
  };
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of(b);
  int64_t before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) s_sum[warp] = before;
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;
  before -= mine;
  int64_t total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  total *= a.kv;
  const int64_t length = max((total + gridDim.x - 1) / gridDim.x, (int64_t)1), from = length * blockIdx.x;
  const int64_t mine_tiles = max((int64_t)0, min(length, total - from));
  for (int b = b0; b < b1; ++b) {
    const int64_t t = tiles_of(b);
    if (mine_tiles > 0 && from >= before * a.kv && from < (before + t) * a.kv) s_seq = b, s_off = from - before * a.kv;
    before += t;
  }
  __syncthreads();
  Run run;
  run.start(a, max(s_seq, 0), mine_tiles > 0 ? s_off : 0, mine_tiles);

  auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
    if (tc::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = tc::globaltimer_ns();
    while (!tc::mbar_try_wait(bar, parity))
      if (abort_flag || tc::globaltimer_ns() - t0 > 2000000000ull) {
        if (a.err) atomicCAS(a.err, 0, 420 + site);
        abort_flag = 1;
        return false;
      }
    return true;
  };

  if (warp == 0 || warp >= 2 + 4 * kGroups) {
    // ------------------------------------------------------------ TMA producers
    const int producer = warp == 0 ? 0 : warp - 1 - 4 * kGroups;
    const int rows = min(a.page, kTile);  // entries per box
    // this lane's box of every key tile: a page's entries, 64 elements of the head
    const int box = lane * kProducers + producer, at = box / (D / 64) * rows, block = box % (D / 64);
    const bool mine = at < kTile;
    // Keys are read once per pass and leave L2 first; the queries and the masses between them stay
    // (131072 entries x 8 heads: 121 -> 112 us; asking for part of the keys to stay for pass 2: 117).
    const uint64_t first = policy_first(), last = policy_last();
    uint32_t kt = 0, qt = 0;
    bool ok = true;
    auto load_queries = [&](int b, int h, int rt) -> bool {
      const uint32_t s = qt % S::kQueries, r = qt / S::kQueries;
      if (r > 0 && !__all_sync(0xffffffffu, wait(&q_empty[s], (r - 1) & 1, 1))) return false;
      ++qt;
      if (lane == 0) {
        tc::mbar_expect_tx(&q_full[s], a.nw * a.groups * D * 2);
        for (int i = 0; i < D / 64; ++i)
          tma_load_5d(queries + s * S::kBytes + i * S::kBlock, &mq, &q_full[s], 0, i, h * a.groups, a.w0 + rt * a.nw, b,
                      last);
      }
      return true;
    };
    // the page of this lane's box in tile t (-1 past the length: zeros); read a tile ahead, since
    // a load from the table takes as long as an SM's share of a tile
    auto page_id = [&](const Run& r, int t) {
      const int e = t * kTile + at;
      return mine && e < r.n ? a.table[r.b * a.table_stride + (e >> a.log_page)] : -1;
    };
    int id = run.left > 0 ? page_id(run, run.t) : -1;
    while (ok && run.left > 0) {
      if (ONE && producer == 0) ok = load_queries(run.b, run.h, 0);
      const Run head = run;
      run.next(a);
      for (int i = 0; ok && i < head.count; ++i) {
        const int now = id, e = (head.t + i) * kTile + at;
        if (i + 1 < head.count) id = page_id(head, head.t + i + 1);
        else if (run.left > 0) id = page_id(run, run.t);
        const uint32_t s = kt % S::kKeys, r = kt / S::kKeys;
        if (r > 0 && !__all_sync(0xffffffffu, wait(&k_empty[s], (r - 1) & 1, 2))) {
          ok = false;
          break;
        }
        ++kt;
        // (another producer's boxes may land first: the phase ends only after this arrival)
        if (producer == 0 && lane == 0) tc::mbar_expect_tx(&k_full[s], S::kBytes);
        if (mine)
          tma_load_5d(keys + s * S::kBytes + block * S::kBlock + at * 128, &mk, &k_full[s], 0, e & (a.page - 1), block, head.h,
                      now, first);
        for (int rt = 0; ok && !ONE && producer == 0 && rt < a.tiles; ++rt) ok = load_queries(head.b, head.h, rt);
      }
    }
    // the loads issued here land before the CTA's shared memory is given up (a key tile's phase ends
    // when both producers' have)
    if (lane == 0) {
      for (uint32_t i = kt > S::kKeys ? kt - S::kKeys : 0; i < kt; ++i) {
        const paged::RingWait w = paged::ring_wait(i, S::kKeys);
        tc::mbar_wait(&k_full[w.stage], w.parity, 200000000ull);
      }
      for (uint32_t i = qt > S::kQueries ? qt - S::kQueries : 0; i < qt; ++i) {
        const paged::RingWait w = paged::ring_wait(i, S::kQueries);
        tc::mbar_wait(&q_full[w.stage], w.parity, 200000000ull);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t fmt = F16 ? 0u : 1u;
      const int n = PASS == 1 ? kTile : (a.nw * a.groups + 15) / 16 * 16;
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
      // the descriptors of the rings' first stages; a stage and a K step add to the address field
      // (bits 0-13, 16-byte units)
      const uint64_t k_desc = tc::sdesc_sw128(tc::smem_u32(keys), 16, 1024);
      const uint64_t q_desc = tc::sdesc_sw128(tc::smem_u32(queries), 16, 1024);
      uint32_t kt = 0, ks = 0, k_phase = 0, qs = 0, q_phase = 0;
      bool ok = true;
      for (; ok && run.left > 0; run.next(a)) {
        if (ONE) ok = wait(&q_full[0], q_phase, 4);
        for (int left = run.count; ok && left > 0; --left, ++kt) {
          ok = wait(&k_full[ks], k_phase, 3);
          for (int rt = 0; ok && rt < a.tiles; ++rt) {
            if (!ONE && !(ok = wait(&q_full[qs], q_phase, 4))) break;
            const uint32_t buf = kt % kGroups, u = kt / kGroups * a.tiles + rt;  // the group's u-th product
            if (u >= 1 && !(ok = wait(&s_empty[buf], (u - 1) & 1, 5))) break;
            tc::fence_after_sync();
            const uint64_t kd0 = k_desc + ks * (S::kBytes >> 4), qd0 = q_desc + qs * (S::kBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t off = ((kk >> 2) * S::kBlock + (kk & 3) * 32) >> 4;
              tc::mma_f16(tmem + buf * kTile, PASS == 1 ? qd0 + off : kd0 + off, PASS == 1 ? kd0 + off : qd0 + off, idesc,
                          kk != 0);
            }
            tc::mma_commit(&s_full[buf]);
            if (!ONE) {
              tc::mma_commit(&q_empty[qs]);
              if (++qs == S::kQueries) qs = 0, q_phase ^= 1;
            }
          }
          if (ok) tc::mma_commit(&k_empty[ks]);
          if (++ks == S::kKeys) ks = 0, k_phase ^= 1;
        }
        if (ONE && ok) {
          tc::mma_commit(&q_empty[0]);
          q_phase ^= 1;
        }
      }
      tc::mma_commit(&drain);  // every MMA issued here completes before the CTA exits
      tc::mbar_wait(&drain, 0, 200000000ull);
    }
  } else {
    // ------------------------------------------------------------ the epilogue groups
    const int group = (warp - 2) >> 2, quad = warp & 3, me = quad * 32 + lane;  // a row (pass 1) or an entry (pass 2)
    const int et = tid - 64;                                                 // 0 .. kEpilogue - 1
    const int rows = a.tiles * kTile;
    uint32_t kt = 0, used = 0;
    bool ok = true;
    auto take = [&](uint32_t& taddr) -> bool {  // the group's next accumulator
      if (!__all_sync(0xffffffffu, wait(&s_full[group], used & 1, 6))) return false;
      tc::fence_after_sync();
      taddr = tmem + ((uint32_t)(quad * 32) << 16) + group * kTile;
      return true;
    };
    auto give = [&]() {
      tc::fence_before_sync();
      tc::mbar_arrive(&s_empty[group]);
      ++used;
    };
    // the place in the sequence of row r of the launch: its token's entry; -1 when it has none
    auto place = [&](int r) {
      const int w = r / kTile * a.nw + r % kTile / a.groups;
      return r % kTile < a.nw * a.groups && a.w0 + w < a.queries ? max(run.n - a.queries + a.w0 + w, -1) : -1;
    };
    for (; run.left > 0; run.next(a)) {
      const int64_t head = (int64_t)run.b * a.kv + run.h;
      float2 ml = make_float2(-INFINITY, 0.f);  // pass 1, ONE: this thread's row
      if (PASS == 1) {
        if (!ONE)
          for (int r = et; r < kGroups * rows; r += kEpilogue) s_stat[r / rows][r % rows] = ml;
        group_sync();
      } else {
        group_sync();  // the last head's logarithms have been read
        // the runs that hold this head, from its first tile in the line
        const int64_t first = from + mine_tiles - run.left - run.t;
        const int run0 = (int)(first / length), run1 = (int)((first + run.tiles - 1) / length);
        for (int r = et; r < rows; r += kEpilogue) {
          float lse = -INFINITY;
          if (place(r) >= 0) {
            if (run0 == run1) {
              lse = a.lse[head * rows + r];
            } else {
              float top = -INFINITY, sum = 0.f;
              for (int i0 = run0; i0 <= run1; i0 += 8) {  // eight pieces' loads in flight
                float2 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const int i = min(i0 + k, run1);
                  x[k] = a.part[((int64_t)i * 2 + (i == run0 ? 1 : 0)) * rows + r];
                  if (i0 + k > run1) x[k] = make_float2(-INFINITY, 0.f);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float up = fmaxf(top, x[k].x);
                  sum = sum * ex2((top - finite(up)) * a.c) + x[k].y * ex2((x[k].x - finite(up)) * a.c);
                  top = up;
                }
              }
              lse = finite(top) * a.c + log2f(sum);
            }
          }
          s_lse[r] = lse == -INFINITY ? -INFINITY : -lse;  // a row without weight adds 0
          s_place[r] = place(r);
        }
        group_sync();
      }
      int id = -1;  // pass 2: the page of this thread's entry, read a turn of the group ahead
      auto page_id = [&](int i) {
        if (PASS == 1 || i >= run.count) return -1;
        const int e = (run.t + i) * kTile + me;
        return e < run.n ? paged::page_of(a.table + run.b * a.table_stride, e, a.log_page, a.pages) : -1;
      };
      id = page_id((int)((group - kt) % kGroups));  // its first tile of this head
      for (int i = 0; ok && i < run.count; ++i, ++kt) {
        if ((int)(kt % kGroups) != group) continue;
        const int t = (run.t + i), e0 = t * kTile;
        const bool whole = e0 + kTile <= run.n - a.queries + 1;  // every row with a place sees all of the tile
        float* to = nullptr;
        float have = 0.f;
        if (PASS == 2) {
          if (id >= 0) {
            to = a.mass + id * a.meta_page + run.h * a.meta_head + ((e0 + me) & (a.page - 1));
            have = *to;
          }
          id = page_id(i + kGroups);
        }
        if (PASS == 1) {
          for (int rt = 0; rt < a.tiles; ++rt) {
            uint32_t taddr;
            if (!(ok = take(taddr))) break;
            const int end_col = whole ? kTile : min(kTile, place(rt * kTile + me) + 1 - e0);  // columns the row sees
            if (!ONE) ml = s_stat[group][rt * kTile + me];
            const uint64_t c2 = pack2(a.c, a.c);
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {  // 64 columns at a time
              uint32_t x[2][32];
#pragma unroll
              for (int i = 0; i < 2; ++i) tc::tmem_ld_32x32(taddr + 64 * half + 32 * i, x[i]);
#pragma unroll
              for (int i = 0; i < 2; ++i) landed(x[i]);
              if (half == 1) give();
              if (!whole)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                  for (int j = 0; j < 32; ++j)
                    if (64 * half + 32 * i + j >= end_col) x[i][j] = 0xff800000u;  // -inf
              float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int j = 0; j < 32; j += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  top[i] = fmaxf(fmaxf(top[i], __uint_as_float(x[i & 1][j + (i >> 1)])),
                                 __uint_as_float(x[i & 1][j + 2 + (i >> 1)]));
              const float up = fmaxf(ml.x, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))), mc = finite(up) * a.c;
              const uint64_t d2 = pack2(-mc, -mc), d[8] = {d2, d2, d2, d2, d2, d2, d2, d2};
              uint64_t sum[4] = {0, 0, 0, 0};  // pairs of zeros
#pragma unroll
              for (int i = 0; i < 4; ++i) add_exps(sum, x[i / 2] + 16 * (i & 1), c2, d);
              const float2 part = unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
              ml.y = ml.y * ex2((ml.x - finite(up)) * a.c) + (part.x + part.y);
              ml.x = up;
            }
            if (!ONE) s_stat[group][rt * kTile + me] = ml;
          }
        } else {
          uint64_t sum[4] = {0, 0, 0, 0};  // pairs of zeros
          const uint64_t c2 = pack2(a.c, a.c);
          for (int rt = 0; rt < a.tiles; ++rt) {
            uint32_t taddr;
            if (!(ok = take(taddr))) break;
            const int valid = min(a.nw, a.queries - a.w0 - rt * a.nw) * a.groups;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (32 * i >= valid) break;
              uint32_t x[32];
              tc::tmem_ld_32x32(taddr + 32 * i, x);
              landed(x);
              const ulonglong2* d4 = reinterpret_cast<const ulonglong2*>(s_lse + rt * kTile + 32 * i);
              const int* at = s_place + rt * kTile + 32 * i;
              if (whole && 32 * i + 32 <= valid) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  uint64_t d[8];
#pragma unroll
                  for (int k = 0; k < 4; ++k) d[2 * k] = d4[4 * j + k].x, d[2 * k + 1] = d4[4 * j + k].y;
                  add_exps(sum, x + 16 * j, c2, d);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  const float w = ex2(__uint_as_float(x[j]) * a.c + s_lse[rt * kTile + 32 * i + j]);
                  sum[j & 3] = add2(sum[j & 3], pack2(e0 + me <= at[j] ? w : 0.f, 0.f));
                }
              }
            }
            give();
          }
          if (!ok) break;
          const float2 part = unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
          if (to != nullptr) *to = have + (part.x + part.y);
        }
      }
      if (PASS == 1) {
        if (ONE)
          for (int i = 0; i < kGroups; ++i) {
            if (group == i) {
              const float2 x = i == 0 ? make_float2(-INFINITY, 0.f) : s_stat[0][me];
              const float up = fmaxf(x.x, ml.x);
              s_stat[0][me] = make_float2(up, x.y * ex2((x.x - finite(up)) * a.c) + ml.y * ex2((ml.x - finite(up)) * a.c));
            }
            group_sync();
          }
        else
          group_sync();
        float2* part = a.part + ((int64_t)blockIdx.x * 2 + (run.t == 0 ? 1 : 0)) * rows;
        for (int r = et; r < rows; r += kEpilogue) {
          constexpr int kSets = ONE ? 1 : kGroups;
          float up = -INFINITY, sum = 0.f;
#pragma unroll
          for (int i = 0; i < kSets; ++i) up = fmaxf(up, s_stat[i][r].x);
#pragma unroll
          for (int i = 0; i < kSets; ++i) sum += s_stat[i][r].y * ex2((s_stat[i][r].x - finite(up)) * a.c);
          if (run.count == run.tiles) a.lse[head * rows + r] = finite(up) * a.c + log2f(sum);
          else part[r] = make_float2(up, sum);
        }
        group_sync();
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) tc::tmem_dealloc(tmem, kTmemCols);
}

constexpr size_t align256(size_t x) { return (x + 255) / 256 * 256; }

struct Plan {
  int groups, nw, row_tiles, ctas;  // row tiles of the whole call
  size_t lse, bytes;
};

Plan make_plan(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_observe_desc& d) {
  Plan p;
  p.groups = d.h / c.kv;
  p.nw = kTile / p.groups < d.queries ? kTile / p.groups : d.queries;
  p.row_tiles = (d.queries + p.nw - 1) / p.nw;
  const int64_t tiles = ((int64_t)b.width * c.page + kTile - 1) / kTile * b.batch * c.kv;
  const int sms = paged_sm_count();
  p.ctas = (int)(tiles < 1 ? 1 : tiles < sms ? tiles : sms);
  const int rows = (p.row_tiles < kMaxTiles ? p.row_tiles : kMaxTiles) * kTile;
  p.lse = align256((size_t)p.ctas * 2 * rows * sizeof(float2));
  p.bytes = p.lse + align256((size_t)b.batch * c.kv * rows * sizeof(float));
  return p;
}

template <int D, bool F16, bool ONE, int PASS>
cudaError_t launch_pass(const ObserveArgs& a, int ctas, const CUtensorMap& mq, const CUtensorMap& mk, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  auto* kernel = paged_observe_kernel<D, F16, ONE, PASS>;
  const cudaError_t e = paged_allow_smem((const void*)kernel, Shape<D, ONE>::kSmem, done);
  if (e != cudaSuccess) return e;
  return launch_after(kernel, dim3((unsigned)ctas), dim3(kThreads), Shape<D, ONE>::kSmem, st, 1, mq, mk, a);
}

template <int D, bool F16, bool ONE>
cudaError_t launch_passes(const ObserveArgs& a, int ctas, const CUtensorMap& mq, const CUtensorMap& mk, cudaStream_t st) {
  const cudaError_t e = launch_pass<D, F16, ONE, 1>(a, ctas, mq, mk, st);
  return e != cudaSuccess ? e : launch_pass<D, F16, ONE, 2>(a, ctas, mq, mk, st);
}

template <int D, bool F16>
cudaError_t launch(const ObserveArgs& a, int ctas, const CUtensorMap& mq, const CUtensorMap& mk, cudaStream_t st) {
  return a.tiles == 1 ? launch_passes<D, F16, true>(a, ctas, mq, mk, st)
                      : launch_passes<D, F16, false>(a, ctas, mq, mk, st);
}

}  // namespace

size_t paged_observe_workspace(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_observe_desc& d) {
  return make_plan(c, b, d).bytes;
}

cudaError_t launch_paged_observe(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_observe_desc& d,
                                 void* ws, cudaStream_t st) {
  const Plan p = make_plan(c, b, d);
  ObserveArgs a = {};
  a.table = b.block_table, a.table_stride = b.table_stride, a.lengths = b.lengths;
  a.batch = b.batch, a.width = b.width, a.page = c.page, a.log_page = paged_log2(c.page), a.pages = c.pages;
  a.kv = c.kv, a.groups = p.groups, a.queries = d.queries, a.nw = p.nw;
  a.c = d.scale * 1.4426950408889634f;
  a.mass = c.mass, a.meta_page = c.meta_page, a.meta_head = c.meta_head;
  a.part = static_cast<float2*>(ws);
  a.lse = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.lse);
  a.err = device_error_word();
  CUtensorMap mq, mk;
  const uint64_t blocks = (uint64_t)(c.d / 64);
  // queries [64 elements][64-element blocks][heads][queries][sequences]; box: the heads of a key head x nw queries
  const uint64_t q_dims[5] = {64, blocks, (uint64_t)d.h, (uint64_t)d.queries, (uint64_t)b.batch};
  const uint64_t q_strides[4] = {128, d.h > 1 ? (uint64_t)d.q_stride_h * 2 : 512,  // of one element: any
                                 d.queries > 1 ? (uint64_t)d.q_stride_t * 2 : 512, b.batch > 1 ? (uint64_t)d.q_stride_b * 2 : 512};
  const uint32_t q_box[5] = {64, 1, (uint32_t)p.groups, (uint32_t)p.nw, 1};
  // keys [64 elements][entries of a page][64-element blocks][heads][pages]; box: the entries of a page (at most 128)
  const uint64_t k_dims[5] = {64, (uint64_t)c.page, blocks, (uint64_t)c.kv, (uint64_t)c.pages};
  const uint64_t k_strides[4] = {(uint64_t)c.stride_entry * 2, 128, (uint64_t)c.stride_head * 2,
                                 (uint64_t)c.stride_page * 2};
  const uint32_t k_box[5] = {64, (uint32_t)(c.page < kTile ? c.page : kTile), 1, 1, 1};
  if (!make_tmap_bf16_sw128(&mq, d.q, 5, q_dims, q_strides, q_box) ||
      !make_tmap_bf16_sw128(&mk, c.k_pages, 5, k_dims, k_strides, k_box))
    return cudaErrorInvalidValue;
  const bool f16 = c.dtype == PBK_F16;
  for (int t = 0; t < p.row_tiles; t += kMaxTiles) {
    a.w0 = t * p.nw;
    a.tiles = p.row_tiles - t < kMaxTiles ? p.row_tiles - t : kMaxTiles;
    cudaError_t e;
    if (c.d == 64) e = f16 ? launch<64, true>(a, p.ctas, mq, mk, st) : launch<64, false>(a, p.ctas, mq, mk, st);
    else if (c.d == 128) e = f16 ? launch<128, true>(a, p.ctas, mq, mk, st) : launch<128, false>(a, p.ctas, mq, mk, st);
    else e = f16 ? launch<256, true>(a, p.ctas, mq, mk, st) : launch<256, false>(a, p.ctas, mq, mk, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace pbk
