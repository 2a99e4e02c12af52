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

__global__ void __launch_bounds__(256)
    paged_move_kernel(const pbk_paged_cache c, const pbk_paged_batch b, const int32_t* src, const int32_t* dst,
                      const int32_t* count, int moves, int log_page) {
  paged::launch_next();
  paged::wait_previous();
  const int h = blockIdx.y, s = blockIdx.z;
  const int64_t row = (int64_t)s * c.kv + h;
  const int n = min(count[row], moves);
  const int chunks = c.d >> 3;
  const int32_t* table = b.block_table + s * b.table_stride;
  const int64_t cap = (int64_t)b.width << log_page;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n * chunks; i += gridDim.x * blockDim.x) {
    const int ch = i % chunks, j = i / chunks;
    const int from = src[row * moves + j], to = dst[row * moves + j];
    if (from < 0 || to < 0 || from >= cap || to >= cap) continue;
    const int fp = paged::page_of(table, from, log_page, c.pages), tp = paged::page_of(table, to, log_page, c.pages);
    if (fp < 0 || tp < 0) continue;
    const int fr = from & (c.page - 1), tr = to & (c.page - 1);
    const int64_t f = fp * c.stride_page + h * c.stride_head + fr * c.stride_entry + 8 * ch;
    const int64_t t = tp * c.stride_page + h * c.stride_head + tr * c.stride_entry + 8 * ch;
    uint16_t* k = reinterpret_cast<uint16_t*>(c.k_pages);
    uint16_t* v = reinterpret_cast<uint16_t*>(c.v_pages);
    *reinterpret_cast<uint4*>(k + t) = *reinterpret_cast<const uint4*>(k + f);
    *reinterpret_cast<uint4*>(v + t) = *reinterpret_cast<const uint4*>(v + f);
    if (ch == 0) {
      const int64_t fm = fp * c.meta_page + h * c.meta_head + fr, tm = tp * c.meta_page + h * c.meta_head + tr;
      if (c.mass != nullptr) c.mass[tm] = c.mass[fm];
      if (c.pos != nullptr) c.pos[tm] = c.pos[fm];
    }
  }
}

// The order of the choice as an unsigned key: protected, then NaN, then the mass downwards.
__device__ __forceinline__ uint32_t select_key(float mass, int pos, int sinks, int64_t first_recent) {
  if ((pos >= 0 && pos < sinks) || pos >= first_recent) return 0xFFFFFFFFu;
  if (mass != mass) return 0xFFFFFFFEu;
  const uint32_t u = __float_as_uint(mass == 0.f ? 0.f : mass);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kSelThreads = 1024;

// One CTA per (sequence, key head): a radix select of the budget-th key, eight bits at a time,
// then one pass in entry order that ranks the free places and the kept entries past the budget.
__global__ void __launch_bounds__(kSelThreads)
    paged_select_kernel(const pbk_paged_cache c, const pbk_paged_batch b, int budget, int recent, int sinks,
                        int32_t* src, int32_t* dst, int32_t* count, int moves, int log_page) {
  paged::launch_next();
  paged::wait_previous();
  const int h = blockIdx.x, s = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t orow = (int64_t)s * c.kv + h;
  int32_t* osrc = src + orow * moves;
  int32_t* odst = dst + orow * moves;
  const int n = paged::clamp_length(b.lengths[s], b.width, c.page);
  const int32_t* table = b.block_table + s * b.table_stride;
  const int64_t first_recent = (int64_t)b.seen[s] - recent;
  int done = 0;
  if (n > budget) {
    auto key_of = [&](int j) -> uint32_t {
      const int page = paged::page_of(table, j, log_page, c.pages);
      float m = 0.f;
      int p = -1;
      if (page >= 0) {
        const int64_t at = page * c.meta_page + h * c.meta_head + (j & (c.page - 1));
        m = c.mass[at];
        p = c.pos[at];
      }
      return select_key(m, p, sinks, first_recent);
    };
    __shared__ uint32_t hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    if (tid == 0) s_prefix = 0, s_need = budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t prefix = s_prefix;
      const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
      for (int j = tid; j < n; j += kSelThreads) {
        const uint32_t key = key_of(j);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        int need = s_need, bin = 255;
        while (bin > 0 && (int)hist[bin] < need) need -= hist[bin--];
        s_need = need;
        s_prefix = prefix | ((uint32_t)bin << shift);
      }
      __syncthreads();
    }
    const uint32_t bar = s_prefix;  // the budget-th key; s_need of the entries equal to it stay
    const int need = s_need;
    __shared__ int wsum[32];
    int eq_run = 0, hole_run = 0, move_run = 0;
    for (int j0 = 0; j0 < n; j0 += kSelThreads) {
      const int j = j0 + tid;
      const uint32_t key = j < n ? key_of(j) : 0u;
      const bool eq = j < n && key == bar;
      const uint32_t eq_bal = __ballot_sync(0xffffffffu, eq);
      if (lane == 0) wsum[warp] = __popc(eq_bal);
      __syncthreads();
      int before = 0, total = 0;
      for (int w = 0; w < 32; ++w) {
        if (w < warp) before += wsum[w];
        total += wsum[w];
      }
      __syncthreads();
      const int eq_rank = eq_run + before + __popc(eq_bal & ((1u << lane) - 1u));
      const bool kept = j < n && (key > bar || (eq && eq_rank < need));
      eq_run += total;
      const bool hole = j < budget && !kept, mover = j >= budget && kept;
      const uint32_t h_bal = __ballot_sync(0xffffffffu, hole), m_bal = __ballot_sync(0xffffffffu, mover);
      if (lane == 0) wsum[warp] = __popc(h_bal) | (__popc(m_bal) << 16);
      __syncthreads();
      before = total = 0;
      for (int w = 0; w < 32; ++w) {
        if (w < warp) before += wsum[w];
        total += wsum[w];
      }
      __syncthreads();
      const uint32_t below = (1u << lane) - 1u;
      if (hole) odst[hole_run + (before & 0xFFFF) + __popc(h_bal & below)] = j;
      if (mover) osrc[move_run + (before >> 16) + __popc(m_bal & below)] = j;
      hole_run += total & 0xFFFF;
      move_run += total >> 16;
    }
    done = hole_run;
  }
  if (tid == 0) count[orow] = done;
  for (int i = done + tid; i < moves; i += kSelThreads) osrc[i] = odst[i] = -1;
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

size_t paged_select_workspace(const pbk_paged_cache&, const pbk_paged_batch&, int) { return 0; }

cudaError_t launch_paged_select(const pbk_paged_cache& c, const pbk_paged_batch& b, int budget, int recent, int sinks,
                                int32_t* src, int32_t* dst, int32_t* count, int moves, void*, cudaStream_t st) {
  return launch_after(paged_select_kernel, dim3(c.kv, b.batch), dim3(kSelThreads), 0, st, 1, c, b, budget, recent, sinks, src,
                      dst, count, moves, paged_log2(c.page));
}

cudaError_t launch_paged_move(const pbk_paged_cache& c, const pbk_paged_batch& b, const int32_t* src,
                              const int32_t* dst, const int32_t* count, int moves, cudaStream_t st) {
  const int64_t blocks = ((int64_t)moves * (c.d / 8) + 255) / 256;
  return launch_after(paged_move_kernel, dim3((unsigned)(blocks < 64 ? blocks : 64), c.kv, b.batch), dim3(256), 0, st, 1, c, b, src,
                      dst, count, moves, paged_log2(c.page));
}

}  // namespace pbk
