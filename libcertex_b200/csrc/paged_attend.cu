// How the attention over a paged cache is split over the GPU, and its launch. The kernels are in paged_attend.cuh, a file per type
// compiles them.
#include "paged_attend.cuh"

#include <algorithm>

namespace certex_b200 {
namespace {

__global__ void take_fault_kernel(int32_t* fault, int32_t* was) { *was = atomicExch(fault, 0); }

/// Shares at most: what the joining kernel's threads read the sums of.
constexpr int64_t kMostShares = kJoinSums * kJoinThreads;
/// Tokens that a block of a cluster goes through at most, as far as the host can tell from the width of the table. Without a split
/// there is one launch and no second pass over partial results, but a block's time is that of the longest row. Rows of 8 KV heads: 1 of
/// 1000 keys 8.3 us in clusters and 9.0 split, 4 of 2000 13.7 and 17.9; with 512 tokens a block 1 of 4000 16.2 and 12.7. Half as many where
/// the clusters leave three quarters of the GPU idle: 1 of 2000 10.9 and 9.4, float32 14.9 and 11.6.
constexpr int64_t kClusterTokens = 256;

/// Shares of a unit, on average, from which blocks have four warps, for 16-bit types and float32. Below that smaller blocks wait less for
/// one another: 128 rows of 100 to 1000 keys took 49 us with four warps and 45 with two (one: 46), one row of 131 072 keys of 8 heads 91.9
/// and 91.3, float32 keys of 16 rows 192 us with four and 175 with one, of one row and 4 KV heads 100 and 90 (131 072) or 39 and 36
/// (40 000). Above, there are too many results to join: one row and KV head of 131 072 keys took 30 us with two warps and 24 with four,
/// two heads of 16 000 float32 keys 18 with one and 15 with four. The same goes for float32 keys with less than 32 tokens to a small
/// block: one row of 2000 keys of 8 heads 12.2 with one and 11.5 with four.
constexpr int64_t kManyShares = 128, kManySharesF32 = 320;

/// Tokens that the table can hold of a sequence, as far as a row may see them.
int64_t table_tokens(const AttendArgs& a)
{
  return std::min(std::min(a.table.pages_per_sequence, kMostTokens) * a.cache.page_size, kMostTokens);
}

struct Plan {
  int32_t per_unit, subs, units, warps;
  int cluster;
  int64_t blocks, shares;
  int part_floats, by_unit, abreast, step_shift;
  size_t bytes;
};

Plan plan_of(const AttendArgs& a, int sm_count)
{
  Plan n;
  const bool half = a.cache.dtype != kPagedF32;
  const int dim   = static_cast<int>(a.cache.head_dim);
  const int group = static_cast<int>(a.n_heads / a.cache.n_kv_heads);
  // a list per query head is a unit of one query; otherwise the heads that share a KV head are taken together
  const bool alone = a.n_lists == a.n_heads && a.n_lists != a.cache.n_kv_heads;
  n.per_unit       = alone ? 1 : std::min(group, half ? 16 : 8);
  n.subs           = (group + n.per_unit - 1) / n.per_unit;
  n.units          = static_cast<int32_t>(a.cache.n_kv_heads) * n.subs;
  int64_t most     = a.n_lists > 0 ? a.k : table_tokens(a);
  if (a.n_lists == 0 && a.window > 0) { most = std::min(most, a.window); }
  const int64_t units = a.n_rows * n.units;
  const int64_t warps    = int64_t(sm_count) * (half ? (dim > 128 ? 4 : n.per_unit <= 8 ? 12 : 8) : 8);  // resident ones
  // as many blocks of four warps per unit as fill the GPU, with 64 tokens each at least
  n.cluster = 1;
  while (n.cluster < 8 && units * n.cluster * 8 <= warps && n.cluster * 64 < most) { n.cluster *= 2; }
  if (most > (units * n.cluster * 16 <= warps ? kClusterTokens / 2 : kClusterTokens) * n.cluster) { n.cluster = 0; }
  const int few          = half ? 2 : 1;  // warps of a small block
  const bool joinable    = half ? warps / few <= kManyShares * units : warps <= kManySharesF32 * units && units * most >= 32 * warps;
  const bool small       = n.cluster ? units * n.cluster * 4 > warps : joinable;
  n.warps                = small ? few : 4;
  const int64_t resident = warps / n.warps;
  // units side by side, where that leaves few blocks without work; lists of positions have no common tokens
  n.abreast = a.n_lists == 0 && n.units <= resident && resident % n.units * 16 <= resident ? n.units : 1;
  // steps are counted in 32 bits
  n.step_shift = kStepShift;
  while (units / n.abreast * ((most >> n.step_shift) + 1 + kLead) >= (int64_t(1) << 30)) { ++n.step_shift; }
  const int64_t steps = (most + (int64_t(1) << n.step_shift) - 1) >> n.step_shift;
  n.shares  = std::min({resident / n.abreast, kMostShares, units / n.abreast * (steps + kLead)});
  n.blocks  = n.cluster ? units * n.cluster : n.shares * n.abreast;
  n.part_floats = n.per_unit * (dim + 4);
  n.bytes       = n.cluster ? 0 : static_cast<size_t>(n.blocks) * 2 * (sizeof(float) * n.part_floats + sizeof(int32_t));
  n.by_unit     = units <= n.blocks;
  return n;
}

/// The largest power of two that divides the strides of pages and tokens in bytes: with 256-byte rows, 32 bits of them reach
/// 1 TB.
int unit_shift(const certexB200PagedCache_t& c)
{
  const int size = paged_type_size(static_cast<int>(c.dtype));
  uint64_t all   = 0;
  for (int i = 0; i < 2; ++i) { all |= static_cast<uint64_t>(c.key_strides[i] * size) | static_cast<uint64_t>(c.value_strides[i] * size); }
  return all == 0 ? 4 : __builtin_ctzll(all);
}

}  // namespace

void paged_divisor(uint32_t d, uint32_t& factor, int32_t& shift)
{
  // with 2^(s-1) < d <= 2^s and m = floor(2^(31 + s) / d) + 1, m d exceeds 2^(31 + s) by e <= d <= 2^s, and floor(n m / 2^(31 + s)) is
  // n / d for all n < 2^31: the excess n e / (d 2^(31 + s)) stays below 1 / d
  shift = 0;
  while ((uint64_t(1) << shift) < d) { ++shift; }
  factor = static_cast<uint32_t>((uint64_t(1) << (31 + shift)) / d + 1);
}

bool paged_within_reach(const certexB200PagedCache_t& c)
{
  const int size  = paged_type_size(static_cast<int>(c.dtype));
  const int shift = unit_shift(c);
  for (const int64_t* s : {c.key_strides, c.value_strides}) {
    if (s[0] < 0 || s[1] < 0) { return false; }
    const double far = static_cast<double>(c.n_pages - 1) * s[0] + static_cast<double>(c.page_size - 1) * s[1];
    if (far * size / (1ull << shift) >= 4294967295.0) { return false; }
  }
  return true;
}

void launch_take_fault(int32_t* fault, int32_t* was, cudaStream_t s) { take_fault_kernel<<<1, 1, 0, s>>>(fault, was); }

size_t paged_attend_workspace(const AttendArgs& a, int sm_count) { return plan_of(a, sm_count).bytes; }

void launch_paged_attend(const AttendArgs& a, int sm_count, cudaStream_t s)
{
  const Plan n = plan_of(a, sm_count);
  AttendParams p{};
  p.keys            = a.cache.keys;
  p.values          = a.cache.values;
  p.unit_shift      = unit_shift(a.cache);
  auto units        = [&](int64_t stride) {
    return static_cast<uint32_t>(stride * paged_type_size(static_cast<int>(a.cache.dtype)) >> p.unit_shift);
  };
  p.k_page          = units(a.cache.key_strides[0]);
  p.k_token         = units(a.cache.key_strides[1]);
  p.k_head          = a.cache.key_strides[2];
  p.v_page          = units(a.cache.value_strides[0]);
  p.v_token         = units(a.cache.value_strides[1]);
  p.v_head          = a.cache.value_strides[2];
  p.n_places        = static_cast<int32_t>(a.cache.n_pages * a.cache.page_size);
  p.n_pages         = static_cast<int32_t>(a.cache.n_pages);
  p.page_size       = static_cast<uint32_t>(a.cache.page_size);
  paged_divisor(p.page_size, p.page_factor, p.page_shift);
  p.dim             = static_cast<int32_t>(a.cache.head_dim);
  p.fault           = a.cache.fault;
  p.pages           = a.table.pages;
  p.page_row        = a.table.row_stride;
  p.n_sequences     = a.table.n_sequences;
  p.most            = static_cast<int32_t>(table_tokens(a));
  p.row_to_sequence = a.table.row_to_sequence;
  p.lengths         = a.lengths;
  p.window          = static_cast<int32_t>(std::min(a.window, kMostTokens));
  p.lists           = a.selected;
  p.lists_64        = a.selected_64;
  p.n_lists         = static_cast<int32_t>(a.n_lists);
  p.k               = static_cast<int32_t>(a.k);
  p.q               = a.q.data;
  p.q_row           = a.q.row_stride;
  p.q_head          = a.q.head_stride;
  const int in_16   = 16 / paged_type_size(static_cast<int>(a.cache.dtype));
  p.q_wide          = reinterpret_cast<uintptr_t>(a.q.data) % 16 == 0 && a.q.row_stride % in_16 == 0 && a.q.head_stride % in_16 == 0;
  p.out             = a.out.data;
  p.o_row           = a.out.row_stride;
  p.o_head          = a.out.head_stride;
  p.lse             = a.lse;
  p.n_rows          = static_cast<int32_t>(a.n_rows);
  p.n_heads         = static_cast<int32_t>(a.n_heads);
  p.group           = static_cast<int32_t>(a.n_heads / a.cache.n_kv_heads);
  p.subs            = n.subs;
  p.per_unit        = n.per_unit;
  p.units           = n.units;
  p.scale           = a.scale * kLog2e;
  p.cluster         = n.cluster;
  p.warps           = n.warps;
  p.step_shift      = n.step_shift;
  p.shares          = static_cast<int32_t>(n.shares);
  p.abreast         = n.cluster ? 1 : n.abreast;
  p.in_line         = n.units / n.abreast;
  p.by_unit         = n.by_unit;
  p.joints          = static_cast<int32_t>(n.by_unit ? a.n_rows * n.units : n.shares * n.abreast);
  const int64_t all = int64_t(p.joints) * n.per_unit;  // queries to be joined
  const bool few    = n.blocks <= 8 * a.n_rows * n.units;  // shares each, on average
  p.join_lanes      = few || all > 4 * sm_count ? 0 : all <= sm_count ? 8 : p.dim <= 128 ? 32 : 64;
  p.part_floats     = n.part_floats;
  p.parts           = static_cast<float*>(a.workspace);
  const bool one    = a.n_lists > 0 || a.n_rows == 1;
  p.marks           = n.cluster || one ? nullptr : reinterpret_cast<int32_t*>(p.parts + 2 * n.blocks * n.part_floats);
  switch (a.cache.dtype) {
    case kPagedF32: return launch_attend_f32(p, n.blocks, s);
    case kPagedF16: return launch_attend_f16(p, n.blocks, s);
    default: return launch_attend_bf16(p, n.blocks, s);
  }
}

}  // namespace certex_b200
