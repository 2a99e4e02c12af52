// The paged cache's bookkeeping: append, eviction choice and moves.
#include "common.cuh"
#include "paged.cuh"

namespace pbk {
namespace {

// One thread per 16-byte chunk of a token's key and value row of one key head.
__global__ void __launch_bounds__(256)
    paged_append_kernel(const pbk_paged_cache c, const pbk_paged_batch b, const uint16_t* k, const uint16_t* v,
                        int64_t stride_t, int64_t stride_h, int tokens, const int32_t* cu, int log_page) {
  paged::launch_next();
  paged::wait_previous();
  const int chunks = c.d >> 3;
  const int64_t work = (int64_t)tokens * c.kv * chunks;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < work; i += (int64_t)gridDim.x * blockDim.x) {
    const int ch = (int)(i % chunks);
    const int64_t th = i / chunks;
    const int h = (int)(th % c.kv), t = (int)(th / c.kv);
    int s = t, at = 0;
    if (cu != nullptr) {  // the sequence whose tokens include t: the last one starting at or before it
      int lo = 0, hi = b.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      s = lo;
      if (t < cu[s] || t >= cu[s + 1]) continue;
      at = t - cu[s];
    }
    const int64_t e = (int64_t)max(b.lengths[s], 0) + at;
    if (e >= (int64_t)b.width << log_page) continue;
    const int page = paged::page_of(b.block_table + s * b.table_stride, (int)e, log_page, c.pages);
    if (page < 0) continue;
    const int row = (int)e & (c.page - 1);
    const int64_t to = page * c.stride_page + h * c.stride_head + row * c.stride_entry + 8 * ch;
    const int64_t from = t * stride_t + h * stride_h + 8 * ch;
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(c.k_pages) + to) = *reinterpret_cast<const uint4*>(k + from);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(c.v_pages) + to) = *reinterpret_cast<const uint4*>(v + from);
    if (ch == 0) {
      const int64_t m = page * c.meta_page + h * c.meta_head + row;
      if (c.mass != nullptr) c.mass[m] = 0.f;
      if (c.pos != nullptr) c.pos[m] = (b.seen != nullptr ? b.seen[s] : max(b.lengths[s], 0)) + at;
    }
  }
}

// A warp takes 8 moves of one (sequence, key head): 8 lanes look up the moves and their pages, then
// all lanes copy the 8 key and value rows, D / 16 16-byte chunks each, every load before the first
// store. Bound by HBM and by how many rows are in flight: a thread per chunk that looks its move
// up itself took 19.1 us for 57344 moves (71 MB).
constexpr int kMoves = 8;            // moves per warp
constexpr int kMoveThreads = 256;

template <int D>
__global__ void __launch_bounds__(kMoveThreads)
    paged_move_kernel(const pbk_paged_cache c, const pbk_paged_batch b, const int32_t* src, const int32_t* dst,
                      const int32_t* count, int moves, int log_page) {
  paged::launch_next();
  paged::wait_previous();
  const int h = blockIdx.y, s = blockIdx.z, lane = threadIdx.x & 31;
  const int64_t row = ((int64_t)s * c.kv + h) * moves;
  const int n = min(count[(int64_t)s * c.kv + h], moves);
  const int first = (blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5)) * kMoves;
  if (first >= n) return;
  // element offsets of this lane's move (lanes below 8), -1 when there is none
  int64_t from = -1, to = -1;
  if (lane < kMoves && first + lane < n) {
    const int fe = src[row + first + lane], te = dst[row + first + lane];
    const int64_t cap = (int64_t)b.width << log_page;
    if (fe >= 0 && te >= 0 && fe < cap && te < cap) {
      const int32_t* table = b.block_table + s * b.table_stride;
      const int fp = paged::page_of(table, fe, log_page, c.pages), tp = paged::page_of(table, te, log_page, c.pages);
      if (fp >= 0 && tp >= 0) {
        const int fr = fe & (c.page - 1), tr = te & (c.page - 1);
        from = fp * c.stride_page + h * c.stride_head + fr * c.stride_entry;
        to = tp * c.stride_page + h * c.stride_head + tr * c.stride_entry;
        const int64_t fm = fp * c.meta_page + h * c.meta_head + fr, tm = tp * c.meta_page + h * c.meta_head + tr;
        if (c.mass != nullptr) c.mass[tm] = c.mass[fm];
        if (c.pos != nullptr) c.pos[tm] = c.pos[fm];
      }
    }
  }
  constexpr int kRow = D / 8, kEach = kMoves * 2 * kRow / 32;  // chunks of a row, chunks per lane
  uint16_t* k = reinterpret_cast<uint16_t*>(c.k_pages);
  uint16_t* v = reinterpret_cast<uint16_t*>(c.v_pages);
  uint4 x[kEach];
  int64_t at[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int chunk = i * 32 + lane, move = chunk / (2 * kRow), r = chunk % (2 * kRow);
    const int64_t f = __shfl_sync(0xffffffffu, from, move);
    at[i] = __shfl_sync(0xffffffffu, to, move);
    if (f >= 0) x[i] = *reinterpret_cast<const uint4*>((r < kRow ? k : v) + f + r % kRow * 8);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = (i * 32 + lane) % (2 * kRow);
    if (at[i] >= 0) *reinterpret_cast<uint4*>((r < kRow ? k : v) + at[i] + r % kRow * 8) = x[i];
  }
}

// The order of the choice as an unsigned key: protected, then NaN, then the mass downwards.
__device__ __forceinline__ uint32_t select_key(float mass, int pos, int sinks, int64_t first_recent) {
  if ((pos >= 0 && pos < sinks) || pos >= first_recent) return 0xFFFFFFFFu;
  if (mass != mass) return 0xFFFFFFFEu;
  const uint32_t u = __float_as_uint(mass == 0.f ? 0.f : mass);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kBins = 2048;          // a digit of 11 bits
// Keys that a CTA keeps in shared memory. With the masks and the histogram 24576 of them are 110 KB,
// so that two CTAs share an SM. Against 32768, one CTA per SM (GPU time, sequences x key heads x
// entries): 60 x 8 x 54806 takes 190 us for 234, 23 x 16 x 198858 756 for 763, but 7 x 16 x 102203
// 53.5 for 50.7. At 23040 heads of 23742 entries are split: 37 x 16 of them take 76 us for 58.
constexpr int kMostKeys = 24576;
constexpr int kMaxCluster = 16;

// Exclusive prefix of x over the CTA's THREADS threads; the sum in *total. Two uses of `scratch`
// need a __syncthreads between them.
template <int THREADS>
__device__ __forceinline__ uint32_t cta_prefix(uint32_t x, uint32_t* scratch, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  if (lane == 31) scratch[warp] = y;
  __syncthreads();
  const uint32_t z = lane < THREADS / 32 ? scratch[lane] : 0u;
  *total = __reduce_add_sync(0xffffffffu, z);
  return __reduce_add_sync(0xffffffffu, lane < warp ? z : 0u) + y - x;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t x;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(x));
  return x;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// A word (four words) of CTA `rank`'s shared memory, at the place that `p` has in this CTA's.
__device__ __forceinline__ uint32_t remote_at(const uint32_t* p, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return at;
}
__device__ __forceinline__ void remote_add(uint32_t* p, uint32_t rank, uint32_t x) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(remote_at(p, rank)), "r"(x) : "memory");
}
__device__ __forceinline__ uint32_t remote(const uint32_t* p, uint32_t rank) {
  uint32_t x;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(remote_at(p, rank)) : "memory");
  return x;
}
__device__ __forceinline__ uint4 remote4(const uint32_t* p, uint32_t rank) {
  uint4 x;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
               : "r"(remote_at(p, rank))
               : "memory");
  return x;
}

// The choice for one (sequence, key head) by a cluster of CTAs, each with an equal share of the
// entries in order, whose keys it computes once and keeps in shared memory (KEEP; longer shares
// compute them again in each pass).
//   1. Three digits of 11, 11 and 10 bits: a histogram of the keys that match the digits so far,
//      summed over the cluster (a CTA owns a part of the bins, the others add theirs to it, all read
//      the sums), from whose top the budget-th key's digit follows.
//   2. Two bit masks per 32 entries: above the budget-th key, and equal to it; of the equal ones
//      the lowest entries of the whole cluster stay until the budget is full.
//   3. Prefix sums over the masks, in the CTA and over the cluster, give every free place below
//      the budget and every kept entry past it its rank in the answer.
// Bound by latency: three histograms and five cluster barriers for a share of some thousand
// entries (8 bytes each), against 1 us for the bytes.
template <int THREADS, bool KEEP>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 4 : 2)
    paged_select_kernel(const pbk_paged_cache c, const pbk_paged_batch b, int budget, int recent, int sinks,
                        int32_t* src, int32_t* dst, int32_t* count, int moves, int log_page, int ctas, int share) {
  extern __shared__ __align__(16) uint32_t smem[];
  uint32_t* hist = smem;                            // [kBins] of this CTA's entries, a digit at a time
  uint32_t* sums = hist + kBins;                    // [3][kBins / ctas] the cluster's, of this CTA's bins; not for one CTA
  uint32_t* masks = sums + (ctas > 1 ? 3 * (kBins / ctas) : 0);  // [share / 32][2]
  uint32_t* keys = masks + share / 16;              // [share], 16-byte aligned: share is a multiple of 64
  __shared__ uint32_t scratch[THREADS / 32], found[2], counts[2];
  paged::launch_next();
  paged::wait_previous();
  const int tid = threadIdx.x, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x / ctas, h = pair % c.kv, s = pair / c.kv;
  const int n = paged::clamp_length(b.lengths[s], b.width, c.page);
  int32_t* osrc = src + (int64_t)pair * moves;
  int32_t* odst = dst + (int64_t)pair * moves;
  if (n <= budget) {  // the whole cluster
    if (rank == 0 && tid == 0) count[pair] = 0;
    for (int i = rank * THREADS + tid; i < moves; i += ctas * THREADS) osrc[i] = odst[i] = -1;
    return;
  }
  const int32_t* table = b.block_table + s * b.table_stride;
  const int64_t first_recent = (int64_t)b.seen[s] - recent;
  // an equal share of 32-entry words per CTA (share is the most, by the table's capacity)
  const int words = (n + 31) / 32, per = (words + ctas - 1) / ctas;
  const int w0 = min((int)rank * per, words), w1 = min(w0 + per, words), e0 = 32 * w0, mine = min(32 * w1, n) - e0;

  // the four keys from entry e0 + i on (i a multiple of 4); past the share's end 0
  auto load_keys = [&](int i) -> uint4 {
    const int e = e0 + i;
    const int id = paged::page_of(table, e, log_page, c.pages), page = max(id, 0);  // no branch between loads
    const int64_t at = page * c.meta_page + h * c.meta_head + (e & (c.page - 1));
    float4 m = *reinterpret_cast<const float4*>(c.mass + at);
    int4 p = *reinterpret_cast<const int4*>(c.pos + at);
    if (id < 0) m = make_float4(0.f, 0.f, 0.f, 0.f), p = make_int4(-1, -1, -1, -1);
    uint4 k;
    k.x = select_key(m.x, p.x, sinks, first_recent);
    k.y = i + 1 < mine ? select_key(m.y, p.y, sinks, first_recent) : 0u;
    k.z = i + 2 < mine ? select_key(m.z, p.z, sinks, first_recent) : 0u;
    k.w = i + 3 < mine ? select_key(m.w, p.w, sinks, first_recent) : 0u;
    return k;
  };
  uint32_t prefix = 0, need = (uint32_t)budget;  // the digits so far; how many of the keys that match them stay
  // Counts a thread's four keys from entry i on (past the share: none) by the digit at `shift`,
  // where they match the digits above it. All lanes of a warp call it together.
  auto count_keys = [&](int shift, int bits, uint4 k, int i) {
    const uint32_t kk[4] = {k.x, k.y, k.z, k.w};
    uint32_t bin[4];
    bool take[4], all = true, any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bin[j] = (kk[j] >> shift) & ((1u << bits) - 1u);
      take[j] = i + j < mine && (shift == 21 || (kk[j] ^ prefix) >> (shift + bits) == 0);
      all = all && take[j] && bin[j] == bin[0];
      any = any || take[j];
    }
    if (!__any_sync(0xffffffffu, any)) return;
    // many entries may share a key (protected ones, those without weight yet): a warp whose 128
    // agree counts them at once
    const uint32_t first = __shfl_sync(0xffffffffu, bin[0], 0);
    if (__all_sync(0xffffffffu, all && bin[0] == first)) {
      if (lane == 0) atomicAdd(&hist[bin[0]], 128u);
    } else if (all) {
      atomicAdd(&hist[bin[0]], 4u);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (take[j]) atomicAdd(&hist[bin[j]], 1u);
    }
  };

  for (int i = tid; i < kBins + (ctas > 1 ? 3 * (kBins / ctas) : 0); i += THREADS) hist[i] = 0;  // and the sums
  if (ctas > 1) cluster_arrive();  // (waited for before anyone adds to another's sums)
  __syncthreads();
  if (KEEP) {
    // the keys into shared memory, the first digit counted on the way; all of a thread's loads of
    // a turn are in flight together
    constexpr int kEach = 4;
    for (int base = 0; base < mine; base += 4 * kEach * THREADS) {
      uint4 k[kEach];
#pragma unroll
      for (int j = 0; j < kEach; ++j) k[j] = load_keys(min(base + 4 * (j * THREADS + tid), (mine - 1) & ~3));
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = base + 4 * (j * THREADS + tid);
        if (i < mine) *reinterpret_cast<uint4*>(keys + i) = k[j];
        count_keys(21, 11, k[j], i);
      }
    }
  }
#pragma unroll 1
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
    if (!KEEP || digit > 0)
      for (int base = 0; base < mine; base += 4 * THREADS) {
        const int i = base + 4 * tid;
        uint4 k = make_uint4(0u, 0u, 0u, 0u);
        if (i < mine) {
          if (KEEP) k = *reinterpret_cast<const uint4*>(keys + i);
          else k = load_keys(i);
        }
        count_keys(shift, bits, k, i);
      }
    __syncthreads();
    // the cluster's sums: bin i is kept by CTA i / (kBins / ctas)
    const int part = kBins / ctas, log_ctas = 31 - __clz(ctas);
    uint32_t* sum_of = sums + digit * part;
    if (ctas > 1) {
      if (digit == 0) cluster_wait();  // every CTA's sums are zero
      for (int i = tid; i < kBins; i += THREADS)
        if (hist[i] != 0) remote_add(sum_of + (i & (part - 1)), i >> (11 - log_ctas), hist[i]);
      cluster_sync();
    }
    // bins from the top, kBins / THREADS per thread; the thread whose bins reach `need` tells
    constexpr int kPer = kBins / THREADS;
    const int low = kBins - kPer * (tid + 1), owner = low >> (11 - log_ctas);
    uint32_t bins[kPer], sum = 0, total;
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const int at = low + kPer - 4 - j;
      const uint4 x = ctas == 1 ? *reinterpret_cast<const uint4*>(hist + at) : remote4(sum_of + (at & (part - 1)), owner);
      bins[j] = x.w, bins[j + 1] = x.z, bins[j + 2] = x.y, bins[j + 3] = x.x;
      sum += (x.x + x.y) + (x.z + x.w);
    }
    uint32_t before = cta_prefix<THREADS>(sum, scratch, &total);
    if (digit < 2)  // (the last digit's counts are read once more below)
      for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
    if (before < need && before + sum >= need) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (before < need && before + bins[j] >= need) {
          found[0] = prefix | ((uint32_t)(low + kPer - 1 - j) << shift);
          found[1] = need - before;
        }
        before += bins[j];
      }
    }
    __syncthreads();
    prefix = found[0], need = found[1];
    __syncthreads();
  }
  // prefix is the budget-th key; `need` of the entries equal to it stay, the lowest first
  const uint32_t equal_before =
      __reduce_add_sync(0xffffffffu, lane < (int)rank ? remote(hist + (prefix & 1023u), lane) : 0u);
  for (int w = tid >> 5; w < w1 - w0; w += (THREADS / 32)) {
    const int i = 32 * w + lane;
    uint32_t k = 0;
    if (i < mine) {
      if (KEEP) {
        k = keys[i];
      } else {
        const uint4 q = load_keys(i & ~3);
        k = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
      }
    }
    const uint32_t gt = __ballot_sync(0xffffffffu, i < mine && k > prefix);
    const uint32_t eq = __ballot_sync(0xffffffffu, i < mine && k == prefix);
    if (lane == 0) masks[2 * w] = gt, masks[2 * w + 1] = eq;
  }
  __syncthreads();
  // a thread per word, in turns: kept entries, then the ranks of free places and movers; the first
  // round counts for the cluster, the second writes
  const int turns = (w1 - w0 + THREADS - 1) / THREADS;
  uint32_t equal_run = equal_before, holes = 0, movers = 0;
  for (int turn = 0; turn < turns; ++turn) {
    const int w = turn * THREADS + tid;
    uint32_t gt = 0, eq = 0, total;
    if (w < w1 - w0) gt = masks[2 * w], eq = masks[2 * w + 1];
    const uint32_t at = equal_run + cta_prefix<THREADS>((uint32_t)__popc(eq), scratch, &total);
    equal_run += total;
    __syncthreads();
    if (w < w1 - w0) {
      const int stay = at >= need ? 0 : min((int)(need - at), __popc(eq));
      uint32_t kept = gt, rest = eq;
      for (int i = 0; i < stay; ++i) kept |= rest & (0u - rest), rest &= rest - 1u;
      // entries below the budget that go, and at or past it that stay
      const int first = e0 + 32 * w;
      const uint32_t exist = n - first >= 32 ? 0xFFFFFFFFu : (1u << (n - first)) - 1u;
      const uint32_t low = budget <= first ? 0u : budget - first >= 32 ? 0xFFFFFFFFu : (1u << (budget - first)) - 1u;
      masks[2 * w] = ~kept & exist & low;
      masks[2 * w + 1] = kept & ~low;
      holes += (uint32_t)__popc(masks[2 * w]), movers += (uint32_t)__popc(masks[2 * w + 1]);
    }
  }
  uint32_t all_holes, all_movers;
  cta_prefix<THREADS>(holes, scratch, &all_holes);
  __syncthreads();
  cta_prefix<THREADS>(movers, scratch, &all_movers);
  if (tid == 0) counts[0] = all_holes, counts[1] = all_movers;
  cluster_sync();
  const uint32_t theirs = lane < ctas ? remote(counts, lane) : 0u, moved = lane < ctas ? remote(counts + 1, lane) : 0u;
  const uint32_t done = __reduce_add_sync(0xffffffffu, theirs);
  uint32_t hole_run = __reduce_add_sync(0xffffffffu, lane < (int)rank ? theirs : 0u);
  uint32_t move_run = __reduce_add_sync(0xffffffffu, lane < (int)rank ? moved : 0u);
  cluster_arrive();  // this CTA has read the others' shared memory for the last time
  uint32_t* ranks = hist;  // of a turn's words: the places their entries take in dst and src
  for (int turn = 0; turn < turns; ++turn) {
    const int first = turn * THREADS, w = first + tid, left = min(w1 - w0 - first, THREADS);
    uint32_t hole = 0, mover = 0, all_h, all_m;
    if (w < w1 - w0) hole = masks[2 * w], mover = masks[2 * w + 1];
    uint32_t hole_at = hole_run + cta_prefix<THREADS>((uint32_t)__popc(hole), scratch, &all_h);
    __syncthreads();
    uint32_t move_at = move_run + cta_prefix<THREADS>((uint32_t)__popc(mover), scratch, &all_m);
    hole_run += all_h, move_run += all_m;
    if (all_h + all_m <= 2u * left) {  // few: each thread writes its word's
      for (; hole != 0; hole &= hole - 1u) odst[hole_at++] = e0 + 32 * w + __ffs(hole) - 1;
      for (; mover != 0; mover &= mover - 1u) osrc[move_at++] = e0 + 32 * w + __ffs(mover) - 1;
    } else {  // many: the words dealt to the warps, a lane per bit, so that neighbours write neighbours
      ranks[2 * tid] = hole_at, ranks[2 * tid + 1] = move_at;
      __syncthreads();
      for (int j = tid >> 5; j < left; j += THREADS / 32) {
        const uint32_t hw = masks[2 * (first + j)], mw = masks[2 * (first + j) + 1], below = (1u << lane) - 1u;
        const int e = e0 + 32 * (first + j) + lane;
        if (hw >> lane & 1u) odst[ranks[2 * j] + __popc(hw & below)] = e;
        if (mw >> lane & 1u) osrc[ranks[2 * j + 1] + __popc(mw & below)] = e;
      }
    }
    __syncthreads();
  }
  if (rank == 0 && tid == 0) count[pair] = (int)done;
  for (int i = (int)done + rank * THREADS + tid; i < moves; i += ctas * THREADS) osrc[i] = odst[i] = -1;
  cluster_wait();  // no CTA leaves while another may read its shared memory
}

}  // namespace

cudaError_t launch_paged_append(const pbk_paged_cache& c, const pbk_paged_batch& b, const void* k, const void* v,
                                int64_t stride_t, int64_t stride_h, int tokens, const int32_t* cu_seqlens,
                                cudaStream_t st) {
  const int64_t work = (int64_t)tokens * c.kv * (c.d / 8);
  const int64_t blocks = (work + 255) / 256;
  return launch_after(paged_append_kernel, dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16)), dim3(256), 0, st, 1, c, b,
                      static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), stride_t, stride_h, tokens,
                      cu_seqlens, paged_log2(c.page));
}

cudaError_t launch_paged_select(const pbk_paged_cache& c, const pbk_paged_batch& b, int budget, int recent, int sinks,
                                int32_t* src, int32_t* dst, int32_t* count, int moves, cudaStream_t st) {
  // CTAs per (sequence, key head): more while a share holds over 2048 entries and the grid has
  // room on the SMs, and as many as it takes to keep the shares in shared memory
  const int64_t pairs = (int64_t)b.batch * c.kv, cap = (int64_t)b.width * c.page;
  int ctas = 1;
  while (ctas < kMaxCluster && ((cap > 2048 * ctas && pairs * 2 * ctas <= 2 * paged_sm_count()) || cap > (int64_t)kMostKeys * ctas))
    ctas *= 2;
  const int64_t words = (cap + 31) / 32, share = ((words + ctas - 1) / ctas + 1) / 2 * 64;
  const bool keep = share <= kMostKeys;
  const int64_t smem = (kBins + (ctas > 1 ? 3 * (kBins / ctas) : 0)) * 4 + share / 4 + (keep ? share * 4 : 0);
  static std::atomic<uint64_t> done[3][2];
  // long shares have more threads, many short ones more CTAs per SM
  const int which = !keep ? 2 : share > 4608 ? 1 : 0;
  auto* kernel = which == 2 ? paged_select_kernel<512, false> : which == 1 ? paged_select_kernel<512, true>
                                                                          : paged_select_kernel<256, true>;
  cudaError_t e = paged_allow((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024, done[which][0]);
  if (e == cudaSuccess && ctas > 8)
    e = paged_allow((const void*)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1, done[which][1]);
  if (e != cudaSuccess) return e;
  pbk_paged_batch used = b;
  if (c.pages == 0) used.width = 0;  // no pages, no entries
  return launch_after(kernel, dim3((unsigned)(pairs * ctas)), dim3(which == 0 ? 256 : 512), (int)smem, st, ctas, c, used,
                      budget, recent, sinks, src, dst, count, moves, paged_log2(c.page), ctas, (int)share);
}

cudaError_t launch_paged_move(const pbk_paged_cache& c, const pbk_paged_batch& b, const int32_t* src,
                              const int32_t* dst, const int32_t* count, int moves, cudaStream_t st) {
  constexpr int kPerBlock = kMoveThreads / 32 * kMoves;
  const dim3 grid((unsigned)(((int64_t)moves + kPerBlock - 1) / kPerBlock), c.kv, b.batch);
  auto* kernel = c.d == 64 ? paged_move_kernel<64> : c.d == 128 ? paged_move_kernel<128> : paged_move_kernel<256>;
  return launch_after(kernel, grid, dim3(kMoveThreads), 0, st, 1, c, b, src, dst, count, moves, paged_log2(c.page));
}

}  // namespace pbk
