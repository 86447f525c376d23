// The operators of a decoding step over a paged cache of keys and values: rotation by position, append, attention of new
// tokens over the cache and over selected positions of it. Definitions in rotate.cu and paged_attend*.cu; the arguments are
// checked by the entry points in c_api.cu.
#pragma once

#include "../../include/certex_b200.h"

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace certex_b200 {

/// Element types of the operators: the kinds of certexB200ToHalf.
enum PagedType : int { kPagedF32 = 0, kPagedF16 = 1, kPagedBF16 = 2 };
inline int paged_type_size(int t) { return t == kPagedF32 ? 4 : 2; }

constexpr int kPagedMaxDim = 256;
constexpr int64_t kMostTokens = (int64_t(1) << 31) - 64;  // that a row may see: tokens are counted in 32 bits

/// y = x turned by `positions` (or back, `inverse`): rows x heads x dim, the first rotary_dim coordinates.
void launch_rotate(const certexB200Rotary_t& plan, const certexB200Rows_t& x, const certexB200Rows_t& y, int64_t n_rows,
                   int64_t n_heads, int64_t head_dim, int dtype, const void* positions, bool positions_64, bool inverse,
                   int sm_count, cudaStream_t s);

/// Keys (turned when `plan` is given) and values to their pages; queries turned into q_out when n_q_heads > 0.
void launch_paged_append(const certexB200PagedCache_t& cache, const certexB200Rotary_t* plan, const certexB200PageTable_t& table,
                         const certexB200Rows_t& k, const certexB200Rows_t& v, const certexB200Rows_t& q,
                         const certexB200Rows_t& q_out, int64_t n_rows, int64_t n_q_heads, const void* positions,
                         bool positions_64, int sm_count, cudaStream_t s);

/// *was = *fault, and *fault = 0.
void launch_take_fault(int32_t* fault, int32_t* was, cudaStream_t s);

/// One call of either attention. `lengths` (with `table`) or `selected` (lists of k physical positions) is given.
struct AttendArgs {
  certexB200PagedCache_t cache;
  certexB200PageTable_t table;
  const int32_t* lengths;
  int64_t window;          // 0: all
  const void* selected;    // [n_rows, n_lists, k], 32 or 64 bits
  int selected_64;
  int64_t n_lists, k;
  certexB200Rows_t q, out;
  int64_t n_rows, n_heads;
  float scale;
  float* lse;              // [n_rows, n_heads] or null
  void* workspace;
};
/// n / d = (2 n * factor >> 32) >> shift for n < 2^31.
void paged_divisor(uint32_t d, uint32_t& factor, int32_t& shift);
/// Whether the kernels' 32-bit offsets, in units that the cache's strides are multiples of, reach all of the cache.
bool paged_within_reach(const certexB200PagedCache_t& cache);
size_t paged_attend_workspace(const AttendArgs& a, int sm_count);
void launch_paged_attend(const AttendArgs& a, int sm_count, cudaStream_t s);

}  // namespace certex_b200
