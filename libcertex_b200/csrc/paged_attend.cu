// Attention of new tokens over a paged cache of keys and values: over the first keys of a sequence
// (certexB200PagedAttend) or over selected positions of the cache (certexB200PagedAttendSelected).
//
//   s_j = scale <q, k_j>,  out = sum_j exp(s_j) v_j / sum_j exp(s_j),  lse = log sum_j exp(s_j)
//
// over the positions j that the row may see; a row that sees none gets zeros and -infinity. Scores, the running maximum m,
// the running sum and the output are held in float32; exp is taken of s_j - m.
#include "paged.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace certex_b200 {
namespace {

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kThreads = 128;

/// A block per (row, head): 128 keys at a time, a thread per key for the scores and per coordinate for the sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) attend_kernel(const AttendArgs a)
{
  __shared__ float q_s[kPagedMaxDim], p_s[kThreads], red[kThreads / 32];
  __shared__ int64_t at_s[kThreads], vat_s[kThreads];
  const int64_t row = blockIdx.x / a.n_heads;
  const int head    = static_cast<int>(blockIdx.x - row * a.n_heads);
  const int dim     = static_cast<int>(a.cache.head_dim);
  const int kv      = static_cast<int>(head / (a.n_heads / a.cache.n_kv_heads));
  const T* q        = static_cast<const T*>(a.q.data) + row * a.q.row_stride + head * a.q.head_stride;
  const T* keys     = static_cast<const T*>(a.cache.keys) + kv * a.cache.key_strides[2];
  const T* values   = static_cast<const T*>(a.cache.values) + kv * a.cache.value_strides[2];
  for (int i = threadIdx.x; i < dim; i += kThreads) { q_s[i] = up(q[i]); }
  int64_t begin = 0, end = a.k, seq = row;
  if (a.lengths) {
    if (a.table.row_to_sequence) { seq = a.table.row_to_sequence[row]; }
    end   = a.lengths[row];
    begin = a.window > 0 && end > a.window ? end - a.window : 0;
    const int64_t most = a.table.pages_per_sequence * a.cache.page_size;
    if (end > 0 && (seq < 0 || seq >= a.table.n_sequences)) { end = 0, *a.cache.fault = 1; }
    if (end > most) { end = most, *a.cache.fault = 1; }
  }
  float m = -INFINITY, total = 0.f, acc[2] = {0.f, 0.f};
  bool any = false;
  for (int64_t t0 = begin; t0 < end; t0 += kThreads) {
    __syncthreads();
    const int64_t t = t0 + threadIdx.x;
    int64_t page = -1, place = 0;
    if (t < end) {
      if (a.lengths) {
        page  = a.table.pages[seq * a.table.row_stride + t / a.cache.page_size];
        place = t % a.cache.page_size;
        if (page < 0 || page >= a.cache.n_pages) { page = -1, *a.cache.fault = 1; }
      } else {
        const int64_t i = (row * a.n_lists + head / (a.n_heads / a.n_lists)) * a.k + t;
        const int64_t p = a.selected_64 ? static_cast<const int64_t*>(a.selected)[i] : static_cast<const int32_t*>(a.selected)[i];
        if (p >= 0) {
          page  = p / a.cache.page_size;
          place = p % a.cache.page_size;
          if (page >= a.cache.n_pages) { page = -1, *a.cache.fault = 1; }
        }
      }
    }
    float s = -INFINITY;
    if (page >= 0) {
      const T* key = keys + page * a.cache.key_strides[0] + place * a.cache.key_strides[1];
      s            = 0.f;
      for (int i = 0; i < dim; ++i) { s += q_s[i] * up(key[i]); }
      s *= a.scale;
    }
    any                = any || __syncthreads_or(page >= 0);
    at_s[threadIdx.x]  = page;
    vat_s[threadIdx.x] = page * a.cache.value_strides[0] + place * a.cache.value_strides[1];
    float top = s;
    for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(~0u, top, o)); }
    if (threadIdx.x % 32 == 0) { red[threadIdx.x / 32] = top; }
    __syncthreads();
    float next = m;
    for (float r : red) { next = fmaxf(next, r); }
    const float base  = next == -INFINITY ? 0.f : next;
    const float alpha = expf(m - base);
    m                 = next;
    const float p     = s != s ? s : expf(s - base);
    p_s[threadIdx.x]  = p;
    __syncthreads();
    total *= alpha, acc[0] *= alpha, acc[1] *= alpha;
    for (int j = 0; j < kThreads; ++j) {
      if (at_s[j] < 0) { continue; }
      total += p_s[j];
      for (int i = 0; i < 2; ++i) {
        const int c = threadIdx.x + i * kThreads;
        if (c < dim) { acc[i] += p_s[j] * up(values[vat_s[j] + c]); }
      }
    }
  }
  T* out = static_cast<T*>(a.out.data) + row * a.out.row_stride + head * a.out.head_stride;
  for (int i = 0; i < 2; ++i) {
    const int c = threadIdx.x + i * kThreads;
    if (c < dim) { put(out + c, any ? acc[i] / total : 0.f); }
  }
  if (a.lse && threadIdx.x == 0) { a.lse[row * a.n_heads + head] = any ? m + logf(total) : -INFINITY; }
}

}  // namespace

size_t paged_attend_workspace(const AttendArgs&, int) { return 0; }

void launch_paged_attend(const AttendArgs& a, int, cudaStream_t s)
{
  const auto grid = static_cast<unsigned>(a.n_rows * a.n_heads);
  if (a.cache.dtype == kPagedF32) {
    attend_kernel<float><<<grid, kThreads, 0, s>>>(a);
  } else if (a.cache.dtype == kPagedF16) {
    attend_kernel<__half><<<grid, kThreads, 0, s>>>(a);
  } else {
    attend_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  }
}

}  // namespace certex_b200
