// The attention weights of a prompt's last queries over the paged cache.
#include "common.cuh"
#include "paged.cuh"

namespace pbk {
namespace {

constexpr int kWarps = 8;

// A maximum over no scores (or over -inf alone) as 0: exp(-inf - 0) is then 0 without a branch,
// and a NaN score stays NaN.
__device__ __forceinline__ float finite(float m) { return m == -INFINITY ? 0.f : m; }

template <bool F16>
__device__ __forceinline__ float2 pair_f32(uint32_t x) {
  if (F16) return __half22float2(*reinterpret_cast<const __half2*>(&x));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}

// One query row (a query head of one token) against the entries [0, end) of a sequence that
// `visible` admits: lane l of a warp holds the dims 2l + 64 i, a warp takes every eighth entry.
struct Rows {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  int64_t sp, se, head;  // strides; the head's offset
  int log_page, pages, pmask;
  __device__ const uint16_t* at(const uint16_t* base, int j) const {
    const int page = paged::page_of(table, j, log_page, pages);
    return page < 0 ? nullptr : base + page * sp + head + (j & pmask) * se;
  }
};

template <bool F16, int D>
__device__ __forceinline__ float dot(const uint16_t* row, const float2 (&q)[D / 64], int lane) {
  float s = 0.f;
  if (row != nullptr)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const float2 x = pair_f32<F16>(*reinterpret_cast<const uint32_t*>(row + 64 * i + 2 * lane));
      s += q[i].x * x.x + q[i].y * x.y;
    }
  return warp_sum(s);
}

template <bool F16, int D>
__device__ __forceinline__ void load_q(const uint16_t* q, float scale, float2 (&out)[D / 64], int lane) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const float2 x = pair_f32<F16>(*reinterpret_cast<const uint32_t*>(q + 64 * i + 2 * lane));
    out[i] = make_float2(x.x * scale, x.y * scale);
  }
}

template <bool F16, int D>
__global__ void __launch_bounds__(32 * kWarps)
    paged_observe_kernel(const pbk_paged_cache c, const pbk_paged_batch b, const pbk_paged_observe_desc a, int log_page) {
  __shared__ float sm_m[kWarps], sm_l[kWarps];
  const int h = blockIdx.x, s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = paged::clamp_length(b.lengths[s], b.width, c.page);
  const int groups = a.h / c.kv;
  const Rows r{static_cast<const uint16_t*>(c.k_pages), nullptr, b.block_table + s * b.table_stride, c.stride_page,
               c.stride_entry, h * c.stride_head, log_page, c.pages, c.page - 1};
  for (int w0 = 0; w0 < a.queries * groups; ++w0) {
    const int w = w0 / groups, j = h * groups + w0 % groups, end = n - a.queries + w + 1;
    if (end <= 0) continue;
    float2 q[D / 64];
    load_q<F16, D>(static_cast<const uint16_t*>(a.q) + s * a.q_stride_b + w * a.q_stride_t + j * a.q_stride_h, a.scale, q, lane);
    float m = -INFINITY, l = 0.f;
    for (int e = warp; e < end; e += kWarps) {
      const float x = dot<F16, D>(r.at(r.k, e), q, lane);
      const float up = fmaxf(m, x);
      l = l * expf(m - finite(up)) + expf(x - finite(up));
      m = up;
    }
    if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sm_m[i]);
    for (int i = 0; i < kWarps; ++i) total += sm_l[i] * expf(sm_m[i] - finite(top));
    if (total != 0.f)
      for (int e = warp; e < end; e += kWarps) {
        const float x = dot<F16, D>(r.at(r.k, e), q, lane);
        const int page = paged::page_of(r.table, e, log_page, c.pages);
        if (lane == 0 && page >= 0)
          c.mass[page * c.meta_page + h * c.meta_head + (e & r.pmask)] += expf(x - (finite(top) + logf(total)));
      }
    __syncthreads();
  }
}

}  // namespace

size_t paged_observe_workspace(const pbk_paged_cache&, const pbk_paged_batch&, const pbk_paged_observe_desc&) { return 0; }

cudaError_t launch_paged_observe(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_observe_desc& d,
                                 void*, cudaStream_t st) {
  const dim3 grid(c.kv, b.batch);
  const int lp = paged_log2(c.page);
  if (c.dtype == PBK_F16) {
    if (c.d == 64) paged_observe_kernel<true, 64><<<grid, 32 * kWarps, 0, st>>>(c, b, d, lp);
    else if (c.d == 128) paged_observe_kernel<true, 128><<<grid, 32 * kWarps, 0, st>>>(c, b, d, lp);
    else paged_observe_kernel<true, 256><<<grid, 32 * kWarps, 0, st>>>(c, b, d, lp);
  } else {
    if (c.d == 64) paged_observe_kernel<false, 64><<<grid, 32 * kWarps, 0, st>>>(c, b, d, lp);
    else if (c.d == 128) paged_observe_kernel<false, 128><<<grid, 32 * kWarps, 0, st>>>(c, b, d, lp);
    else paged_observe_kernel<false, 256><<<grid, 32 * kWarps, 0, st>>>(c, b, d, lp);
  }
  return cudaGetLastError();
}

}  // namespace pbk
