// Attention of new tokens over a paged cache of keys and values: over the first keys of a sequence
// (certexB200PagedAttend) or over selected positions of the cache (certexB200PagedAttendSelected).
//
//   s_j = scale <q, k_j>,  out = sum_j exp(s_j) v_j / sum_j exp(s_j),  lse = log sum_j exp(s_j)
//
// over the positions j that the row may see; a row that sees none gets zeros and -infinity.
//
// What bounds it: every key and value is read once from HBM, for at most a few dozen operations per byte (two products for
// each query head that shares the KV head). So the work is a stream of rows of 2 d bytes from addresses that the page table or
// the list of positions names, and everything else has to fit beside it:
//
//  * One pass. Scores, the running maximum m, the running sum l and the output stay in registers in float32;
//    when m grows, l and the output are multiplied by exp2(m_old - m_new). Scores are kept in units of log2 e, so that a
//    weight is one subtraction and one exp2.
//  * The stream is split evenly. The tokens that all rows of the call see, in steps of 32, are one sequence of work that
//    is cut into equal shares, a share per resident block, wherever the cuts fall: 1 row of 131 072 keys and 64 rows of 1 to
//    8192 keys load the GPU alike, and lengths are read on the device only. A row and KV head ("unit") that
//    a cut divides leaves a partial result (m, l, output) per share, which a second, small kernel joins in the order of the
//    shares: results do not depend on timing. It is launched while the first still runs and waits for it.
//    Calls whose units are known to be short take a block, or a cluster of blocks, per unit and one launch.
//  * A warp works by itself on tiles of 16 or 32 keys, by turns with the W warps of its block: no barrier until a unit ends, and
//    the loads of the next tile are in flight while one is computed. The table's entries for a tile are asked for a tile before
//    its loads, and where it lies is worked out while the tile before it arrives: done between two tiles' products instead, a call
//    over 131 072 keys took 105 us instead of 94, and float32 keys 240 instead of 192.
//
// 131 072 bfloat16 keys of 8 heads of 128: 91 us, 5.9 TB/s; 16 rows of 32 lists of 2048 positions 95 us, 5.1 TB/s. About 11 us of
// either are the launches, the first tile's chain of reads (length, page, row), blocks that end unevenly and the joining; the rest runs
// at 6 to 6.4 TB/s, near the rate of a copy. Asking L2 for rows two tiles ahead made everything slower (a prefetch per row 108 and 160 us
// for these two, one per line 98 and 208): the reads in flight are enough, and DRAM has its own order to keep.
//
// Rows that are not to be seen have scores of -infinity and values of zero, so nothing that lies there (NaN, infinity,
// another sequence's tokens) has an effect.
#pragma once

#include "paged.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace certex_b200 {

/// What the kernels need, in the sizes that they compute with.
struct AttendParams {
  const void* keys;
  const void* values;
  // strides of pages and tokens in units of 2^unit_shift bytes, of heads in elements
  uint32_t k_page, k_token, v_page, v_token;
  int64_t k_head, v_head;
  int32_t unit_shift;
  uint32_t page_factor;  // t / page_size = (2 t * page_factor >> 32) >> page_shift
  int32_t page_shift;
  int32_t n_places;      // n_pages * page_size
  int32_t n_pages;
  uint32_t page_size;
  int32_t dim;
  int32_t* fault;
  // what a row sees
  const int32_t* pages;
  int64_t page_row;
  int64_t n_sequences;
  int32_t most;               // tokens that the table can hold
  const int32_t* row_to_sequence;
  const int32_t* lengths;     // null: lists
  int32_t window;
  const void* lists;
  int32_t lists_64, n_lists;
  int32_t k;
  // queries and answers
  const void* q;
  int64_t q_row, q_head;
  int32_t q_wide;  // every query lies on 16 bytes
  void* out;
  int64_t o_row, o_head;
  float* lse;
  int32_t n_rows;
  int32_t n_heads, group, subs, per_unit;  // query heads per KV head; units per KV head; query heads of a unit
  int32_t units;                           // of a row
  float scale;                             // in units of log2 e
  // the split
  int32_t warps;       // of a block
  int32_t cluster;     // blocks of a unit, in a cluster; 0: the work is split evenly
  int32_t step_shift;  // log2 of the tokens of a step
  int32_t shares;      // that the work is split into at most
  int32_t abreast;     // blocks of a share: 1, or the units of a row
  int32_t in_line;     // units of a row that lie behind one another among the steps: units / abreast
  int32_t by_unit;     // the call has no more units than blocks: the second kernel has blocks per unit, not per block
  // where that follows from one length it finds a unit's shares itself; otherwise (not null) the blocks leave it, [blocks][2]:
  // the unit that a block begins and leaves unfinished, and how many shares it has (0: there is none), or by unit, [units][2]:
  // the share that begins it, and how many it has (0: no more than that)
  int32_t* marks;
  int32_t joints;      // units or blocks that it looks at
  int32_t join_lanes;  // 0: a warp for a joint's query; else its threads that share a partial result, with four coordinates each
  float* parts;        // [blocks][2] partial results of part_floats each
  int32_t part_floats;
};

/// Launches the attention (and the joining of its shares) for rows of one type: float, __half or __nv_bfloat16, a file each.
void launch_attend_f32(const AttendParams& p, int64_t blocks, cudaStream_t s);
void launch_attend_f16(const AttendParams& p, int64_t blocks, cudaStream_t s);
void launch_attend_bf16(const AttendParams& p, int64_t blocks, cudaStream_t s);

namespace {

constexpr int kStepShift = 5;  // the work is cut in steps of 32 tokens (more where 32 bits would not count them)
constexpr int kLead      = 4;  // steps that a unit's beginning and end count for: fetching its first tiles, joining the warps
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2   = 0.6931471805599453f;

// ------------------------------------------------------------------------------------------------ types
template <typename T>
struct Type;
template <>
struct Type<float> {
  static __device__ float down(float v) { return v; }
};
template <>
struct Type<__half> {
  static __device__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Type<__nv_bfloat16> {
  static __device__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ float exp2_fast(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t smem_of(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

/// 16 bytes to shared memory, or 16 zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------------------------------------ what a row sees
struct Span {
  int32_t begin;  // first token
  int32_t count;
  int32_t sequence;
};

/// EARLY: read from L2, before this kernel has waited for the one in front.
template <bool EARLY = false>
__device__ __forceinline__ Span span_of(const AttendParams& p, int32_t row)
{
  if (p.lengths == nullptr) { return {0, p.k, 0}; }
  auto read              = [&](const int32_t* at) { return EARLY ? __ldcg(at + row) : at[row]; };
  int32_t end            = read(p.lengths);
  const int32_t sequence = p.row_to_sequence ? read(p.row_to_sequence) : row;
  if (end <= 0) { return {0, 0, 0}; }
  const bool stranger = sequence < 0 || sequence >= p.n_sequences;
  if (stranger || end > p.most) { *p.fault = 1; }
  if (stranger) { return {0, 0, 0}; }
  end                 = min(end, p.most);
  const int32_t begin = p.window > 0 && end > p.window ? end - p.window : 0;
  return {begin, end - begin, sequence};
}

/// One unit's share: tokens [i0, i1) of what its row sees.
struct Segment {
  int32_t row, kv, head, n_heads;  // KV head, first query head, query heads
  int32_t slot;               // of the partial result, -1: this is the whole unit
  int32_t i0, i1;
  int32_t begin;
  const void* index;          // the sequence's row of the table, or the list
};

__device__ __forceinline__ Segment segment_of(const AttendParams& p, int32_t row, const Span& s, int unit)
{
  Segment g;
  g.row     = row;
  g.kv      = p.subs == 1 ? unit : unit / p.subs;
  const int sub = unit - g.kv * p.subs;
  g.head    = g.kv * p.group + sub * p.per_unit;
  g.n_heads = min(p.per_unit, p.group - sub * p.per_unit);
  g.begin   = s.begin;
  if (p.lengths) {
    g.index = p.pages + s.sequence * p.page_row;
  } else {
    const int64_t list = int64_t(row) * p.n_lists + (p.n_lists == 1 ? 0 : p.n_lists == p.n_heads ? g.head : g.kv);
    g.index            = static_cast<const char*>(p.lists) + list * p.k * (p.lists_64 ? 8 : 4);
  }
  return g;
}

/// Where a key and its value lie, in units from the first key and value of their head; kNowhere for one that is not seen.
struct Place {
  uint32_t k, v;
};
constexpr uint32_t kNowhere = ~0u;

/// Whole pages in t < 2^31 tokens.
__device__ __forceinline__ uint32_t pages_in(const AttendParams& p, uint32_t t) { return __umulhi(2 * t, p.page_factor) >> p.page_shift; }

/// Entry of the table, or of the list, that token i of what a row sees goes by (with the segment's begin and index). Nothing here
/// depends on what is read: the kernels ask for it a tile before they need it.
__device__ __forceinline__ int64_t entry_of(const AttendParams& p, int32_t begin, const void* index, int32_t i)
{
  if (p.lengths) { return static_cast<const int32_t*>(index)[pages_in(p, begin + i)]; }
  return p.lists_64 ? static_cast<const int64_t*>(index)[i] : static_cast<const int32_t*>(index)[i];
}

/// The place of token i from its entry.
__device__ __forceinline__ Place place_of(const AttendParams& p, int32_t begin, int32_t i, int64_t entry)
{
  // its number among the tokens of its sequence, or of the cache
  const uint32_t t = p.lengths ? static_cast<uint32_t>(begin + i) : static_cast<uint32_t>(entry);
  const uint32_t n = pages_in(p, t), place = t - n * p.page_size;
  const uint32_t page = p.lengths ? static_cast<uint32_t>(entry) : n;
  const bool wrong    = p.lengths ? page >= static_cast<uint32_t>(p.n_pages) : entry >= p.n_places;  // (pages: negative ones too)
  if (wrong) { *p.fault = 1; }
  if (wrong || (!p.lengths && entry < 0)) { return {kNowhere, kNowhere}; }
  return {page * p.k_page + place * p.k_token, page * p.v_page + place * p.v_token};
}

// The work of a call that is split: the steps of all units in a row, kLead steps and those of its tokens for every unit that
// sees something, units of a row next to each other. Share w is the steps [first_step(w), first_step(w + 1)).
// Sequences are split with their units side by side instead (`abreast`): a row counts once, and every share belongs to as many
// neighbouring blocks as a row has units, one each. They go through the same tokens at the same time, whose heads lie next to
// one another in memory where the heads are the inner axis.
__device__ __forceinline__ int32_t steps_for(const AttendParams& p, int32_t count)
{
  return count > 0 ? static_cast<int32_t>((static_cast<uint32_t>(count) + (1u << p.step_shift) - 1) >> p.step_shift) + kLead : 0;
}

/// a / b of what is not negative (signed division is a longer chain of instructions).
__device__ __forceinline__ int32_t divide(int32_t a, int32_t b) { return static_cast<uint32_t>(a) / static_cast<uint32_t>(b); }

struct Split {
  int32_t total, shares, each, more;  // the first `more` shares have a step more than `each`
  Split() = default;
  __device__ Split(int32_t steps, int32_t most) : total(steps), shares(min(most, steps)), each(0), more(0)
  {
    if (shares > 0) {
      each = divide(total, shares);
      more = total - each * shares;
    }
  }
  __device__ int32_t first_step(int32_t w) const { return w * each + min(w, more); }
  __device__ int32_t share_of(int32_t step) const
  {
    const int32_t x = more * (each + 1);
    return step < x ? divide(step, each + 1) : more + divide(step - x, each);
  }
};

/// A unit's place among the steps.
struct Unit {
  int32_t row, begin, steps;  // begin: its first step
  int32_t unit;
  Span span;
};

/// The split and where a block's share of it begins; a block of W warps calls it as a whole.
struct Start {
  Split split;
  int32_t at;  // the share's first step
  Unit unit;   // whose steps that is among; undefined when the split has not so many shares
};

template <int W>
__device__ __forceinline__ Start start_of(const AttendParams& p, int32_t share)
{
  constexpr int kThreads = W * 32;
  __shared__ int32_t sums[W];
  __shared__ int32_t found[2];
  __shared__ Span spans;
  const bool alike = !p.lengths || p.n_rows == 1;  // every unit has the same steps
  if (alike) {
    const Span span     = span_of(p, 0);
    const int32_t steps = steps_for(p, span.count), each = steps * p.in_line;
    Start x{Split(p.n_rows * each, p.shares), 0, {0, 0, steps, 0, span}};
    if (share >= x.split.shares) { return x; }
    x.at         = x.split.first_step(share);
    x.unit.row   = p.n_rows == 1 ? 0 : divide(x.at, each);
    const auto u = divide(x.at - x.unit.row * each, steps);
    x.unit.unit  = static_cast<int>(u);
    x.unit.begin = x.unit.row * each + u * steps;
    return x;
  }
  // an inclusive sum over the block for kThreads rows at a time; the total first, where they are more
  if (threadIdx.x == 0) { found[0] = -1; }
  __syncthreads();
  int32_t total = 0;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const bool once = p.n_rows <= kThreads;
  if (!once) {
    int32_t mine = 0;
    for (int32_t row = threadIdx.x; row < p.n_rows; row += kThreads) { mine += steps_for(p, span_of(p, row).count); }
    for (int o = 16; o > 0; o >>= 1) { mine += __shfl_xor_sync(~0u, mine, o); }
    if (lane == 0) { sums[warp] = mine; }
    __syncthreads();
    for (int w = 0; w < W; ++w) { total += sums[w]; }
    __syncthreads();
  }
  Start x{Split(total * p.in_line, p.shares), 0, {}};
  if (!once) { x.at = x.split.first_step(share); }
  int32_t before = 0;
  for (int32_t r0 = 0; r0 < p.n_rows; r0 += kThreads) {
    const int32_t r = r0 + threadIdx.x;
    const Span span = r < p.n_rows ? span_of(p, r) : Span{0, 0, 0};
    const int32_t n = steps_for(p, span.count) * p.in_line;
    int32_t upto    = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t y = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) { upto += y; }
    }
    if (W > 1) {
      if (lane == 31) { sums[warp] = upto; }
      __syncthreads();
    }
    int32_t first = before + upto - n;
    if (W > 1) {
      for (int i = 0; i < W; ++i) {
        if (i < warp) { first += sums[i]; }
        before += sums[i];
      }
    } else {
      before += __shfl_sync(~0u, upto, 31);
    }
    if (once) {
      x.split = Split(before, p.shares);
      x.at    = x.split.first_step(share);
    }
    if (first <= x.at && x.at < first + n) { found[0] = r, found[1] = first, spans = span; }
    if (x.at < before) { break; }
    if (W > 1) { __syncthreads(); }
  }
  __syncthreads();
  if (found[0] < 0) { x.split = Split(0, 0); }  // no share, or lengths that somebody changes meanwhile
  if (share < x.split.shares) {
    x.unit.row   = found[0];
    x.unit.span  = spans;
    x.unit.steps = steps_for(p, spans.count);
    const auto u = divide(x.at - found[1], x.unit.steps);
    x.unit.unit  = static_cast<int>(u);
    x.unit.begin = found[1] + u * x.unit.steps;
  }
  return x;
}

/// The blocks are there before the kernel in front of them has ended (2 us less between calls in a stream) and wait for that; the
/// joining kernel, if there is one, is let in the same way, but never before the wait: it reads what that kernel wrote (joint_of).
__device__ __forceinline__ void begin(const AttendParams& p)
{
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!p.cluster) { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
}

/// Calls body(segment) for this block's share of the work. A block of W warps calls it as a whole.
template <typename T, int W, typename F>
__device__ __forceinline__ void for_segments(const AttendParams& p, F&& body)
{
  constexpr int kThreads = W * 32;
  auto nothing_seen = [&](int32_t row, int head, int n_heads) {
    for (int h = head; h < head + n_heads; ++h) {
      T* o = static_cast<T*>(p.out) + int64_t(row) * p.o_row + h * p.o_head;
      for (int c = threadIdx.x; c < p.dim; c += kThreads) { o[c] = Type<T>::down(0.f); }
      if (p.lse && threadIdx.x == 0) { p.lse[int64_t(row) * p.n_heads + h] = -INFINITY; }
    }
  };
  // What a block works on lies in shared memory: the registers are needed for the work. The first thread of the last warp, which
  // has the fewest tiles, works out the next segment while the others begin with one.
  struct State {
    int32_t at, end;
    Split split;
    Unit u;
  };
  __shared__ Segment segments[2];
  __shared__ State state;
  const int32_t block = blockIdx.x, share = divide(block, p.abreast), beside = block - share * p.abreast;
  auto next = [&](Segment& g) {
    g.n_heads = 0;  // nothing left
    while (state.at < state.end) {
      Unit u           = state.u;
      const int32_t at = state.at, end = state.end, to = min(end, u.begin + u.steps);
      const int32_t i0 = max(0, at - u.begin - kLead) << p.step_shift;
      const auto i1    = static_cast<int32_t>(min(int64_t(u.span.count), int64_t(max(0, to - u.begin - kLead)) << p.step_shift));
      if (i0 < i1) {  // (a share may end within a unit's lead)
        const int unit    = u.unit + beside;
        g                 = segment_of(p, u.row, u.span, unit);
        const bool begins = i0 == 0, ends = i1 == u.span.count;
        g.i0 = i0, g.i1 = i1;
        // a partial result that begins a unit belongs to the block's second slot, one that goes on with it to the first
        g.slot = begins && ends ? -1 : 2 * block + (begins ? 1 : 0);
        if (p.marks && begins && (!ends || p.by_unit)) {
          const int32_t id = u.row * p.units + unit;
          int32_t* mark    = p.marks + 2 * (p.by_unit ? id : block);
          mark[0]          = p.by_unit ? share : id;
          mark[1]          = ends ? 0 : state.split.share_of(u.begin + u.steps - 1) - share + 1;
        }
      }
      if (to < end) {
        u.begin += u.steps;
        if (++u.unit == p.in_line) {
          u.unit = 0;
          do {  // (there are steps left: a row behind has some, unless somebody changes the lengths meanwhile)
            u.span = ++u.row < p.n_rows ? span_of(p, u.row) : Span{0, 0, 0};
          } while (u.span.count == 0 && u.row < p.n_rows);
          u.steps = steps_for(p, u.span.count);
        }
        state.u = u;
      }
      state.at = u.steps > 0 ? to : end;
      if (i0 < i1) { break; }
    }
  };
  constexpr int kScribe = kThreads - 32;
  if (p.cluster) {
    // the blocks of a cluster share a unit's tokens, 16 by 16
    const int32_t unit = divide(block, p.cluster), rank = block - unit * p.cluster, row = divide(unit, p.units);
    const Span s = span_of(p, row);
    Segment g    = segment_of(p, row, s, unit - row * p.units);
    if (s.count == 0) {
      if (rank == 0) { nothing_seen(row, g.head, g.n_heads); }
      return;
    }
    const int32_t tiles = (s.count + 15) / 16;  // (a cluster's rows are short)
    g.i0   = divide(tiles * rank, p.cluster) * 16;
    g.i1   = min(s.count, divide(tiles * (rank + 1), p.cluster) * 16);
    g.slot = -1;
    if (threadIdx.x == kScribe) { segments[0] = g, state.at = state.end = 0; }
  } else {
    // rows that see nothing have no steps: the blocks share them out
    if (p.lengths) {
      for (int32_t row = block; row < p.n_rows; row += gridDim.x) {
        if (span_of(p, row).count == 0) {
          nothing_seen(row, 0, p.n_heads);
          if (p.marks && p.by_unit) {
            for (int u = threadIdx.x; u < p.units; u += kThreads) { p.marks[2 * (row * p.units + u) + 1] = 0; }
          }
        }
      }
    }
    const Start x = start_of<W>(p, share);
    if (p.marks && !p.by_unit && threadIdx.x == kScribe) { p.marks[2 * block + 1] = 0; }
    if (share >= x.split.shares) { return; }
    if (threadIdx.x == kScribe) {
      state.at = x.at, state.end = x.split.first_step(share + 1), state.split = x.split, state.u = x.unit;
      next(segments[0]);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int turn = 0; segments[turn].n_heads > 0; turn ^= 1) {
    if (threadIdx.x == kScribe) { next(segments[turn ^ 1]); }
    body(segments[turn]);  // ends with a barrier
  }
}

/// The answer of a unit's query head from its sums, or a partial result: coordinate c of query i.
template <typename T>
__device__ __forceinline__ void put_out(const AttendParams& p, const Segment& g, int i, int c, float v)
{
  if (g.slot >= 0) {
    p.parts[int64_t(g.slot) * p.part_floats + 4 * p.per_unit + i * p.dim + c] = v;
  } else {
    (static_cast<T*>(p.out) + int64_t(g.row) * p.o_row + (g.head + i) * p.o_head)[c] = Type<T>::down(v);
  }
}

/// m, l and whether anything was seen, of query i (once per query).
__device__ __forceinline__ void put_sums(const AttendParams& p, const Segment& g, int i, float m, float l, bool any)
{
  if (g.slot >= 0) {
    float* to = p.parts + int64_t(g.slot) * p.part_floats + 4 * i;
    to[0] = m, to[1] = l, to[2] = any ? 1.f : 0.f;
  } else if (p.lse) {
    p.lse[int64_t(g.row) * p.n_heads + g.head + i] = any ? (m + log2f(l)) * kLn2 : -INFINITY;
  }
}

// ------------------------------------------------------------------------------------------------ 16-bit types
// Tensor cores by warp-level products (mma.m16n8k16): with one new token there are 1 to 16 queries per KV head, and tcgen05's
// smallest tile of 128 rows would be nearly empty. Keys and values take the 16-row side of the product and the
// queries the 8-column side, so that 8 queries fill it: S^T = K Q^T, then O^T = V^T P^T. The two products of a tile of
// 16 keys by d = 128 are 8 + 16 instructions for 8 KB read.
//
// Weights enter the second product as two 16-bit numbers, the upper part cut off and the rest, because a weight rounded once to
// bfloat16 would add as much error as the rounding of the result. p = hi + lo to 2^-16 of p in bfloat16, in float16 to 2^-20 of p
// and 2^-41 of the row's largest weight so far: float16 has nothing below 2^-24, so its weights are multiplied by 2^16 (l carries
// the factor too, so it cancels). What is cut off is a little less than p, so that neither part of a weight is zero and an infinite
// value stays one (zero times infinity is NaN); a weight of zero is two zeros and adds nothing.
constexpr int kKeys   = 16;  // of a tile
constexpr int kStages = 3;

__device__ __forceinline__ void load_matrix(uint32_t (&a)[4], uint32_t at)
{
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_matrix_t(uint32_t (&a)[4], uint32_t at)
{
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v)
{
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

/// A little less than x, by 2^-20 of it and `least`, a step or two of what is subnormal in the type; 0 for 0 (and for NaN, which the
/// lower part keeps).
__device__ __forceinline__ float below(float x, float least) { return fmaxf(fmaf(x, 1.f - 0x1p-20f, -least), 0.f); }

template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  static constexpr float kRaise = 0.f;  // log2 of the factor on weights
  static __device__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
  {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  /// (x, y) as two pairs of numbers whose sum they are; x in the lower halves.
  static __device__ void split(float x, float y, uint32_t& hi, uint32_t& lo)
  {
    const uint32_t a = __float_as_uint(below(x, 0x1p-132f)) & 0xffff0000u, b = __float_as_uint(below(y, 0x1p-132f)) & 0xffff0000u;
    hi = (a >> 16) | b;
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - __uint_as_float(a), y - __uint_as_float(b));
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <>
struct Half<__half> {
  static constexpr float kRaise = 16.f;  // (the largest weight is cut to 65 504, the largest number)
  static __device__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
  {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ void split(float x, float y, uint32_t& hi, uint32_t& lo)
  {
    const __half2 h = __halves2half2(__float2half_rz(below(x, 0x1p-24f)), __float2half_rz(below(y, 0x1p-24f)));
    hi              = *reinterpret_cast<const uint32_t*>(&h);
    const __half2 r = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    lo              = *reinterpret_cast<const uint32_t*>(&r);
  }
};

/// What the block's warps found of a segment meets in shared memory (`sums`: a warp's [queries][D + 4] floats: output, m, l, seen;
/// `pitch` floats between warps), for a cluster in its first block's reach, and goes out. m is relative to weights that were
/// raised by 2^raise.
template <typename T, int D, int W>
__device__ __forceinline__ void finish_segment(const AttendParams& p, const Segment& g, float* sums, int pitch, float raise)
{
  constexpr int kRow = D + 4, kThreads = W * 32;
  __shared__ float weight[16][W], total[16][4];  // of a query: the warps' factors; m, l, seen
  __shared__ float others[16][8];                      // the factors of a cluster's blocks
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid < g.n_heads) {
    float m[W], top = -INFINITY, sum = 0.f, seen = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      m[x] = sums[x * pitch + tid * kRow + D];
      top  = fmaxf(top, m[x]);
    }
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float* from = sums + x * pitch + tid * kRow + D;
      const float f     = top == -INFINITY ? 1.f : exp2_fast(m[x] - top);
      weight[tid][x]    = f;
      sum += f * from[1];
      seen += from[2];
    }
    total[tid][0] = top, total[tid][1] = sum, total[tid][2] = seen;
    if (p.cluster <= 1) { put_sums(p, g, tid, top - raise, sum, seen > 0.f); }
  }
  __syncthreads();
  if (p.cluster <= 1) {
    for (int i = 0; i < g.n_heads; ++i) {
      const float seen = total[i][2], scale = g.slot >= 0 ? 1.f : 1.f / total[i][1];
      for (int c = tid; c < p.dim; c += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int x = 0; x < W; ++x) { v += weight[i][x] * sums[x * pitch + i * kRow + c]; }
        put_out<T>(p, g, i, c, seen > 0.f ? v * scale : 0.f);
      }
    }
    __syncthreads();
    return;
  }
  // the block's result in the place of its first warp's
  for (int i = 0; i < g.n_heads; ++i) {
    for (int c = tid; c < p.dim; c += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x) { v += weight[i][x] * sums[x * pitch + i * kRow + c]; }
      sums[i * kRow + c] = v;
    }
  }
  const auto cluster = cooperative_groups::this_cluster();
  cluster.sync();
  const int rank = static_cast<int>(cluster.block_rank());
  if (tid < g.n_heads) {
    float top = -INFINITY, sum = 0.f, seen = 0.f;
    float m[8], l[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      if (x < p.cluster) {
        const float* from = cluster.map_shared_rank(&total[tid][0], x);
        m[x] = from[0], l[x] = from[1], seen += from[2];
        top = fmaxf(top, m[x]);
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      if (x < p.cluster) {
        const float f = top == -INFINITY ? 1.f : exp2_fast(m[x] - top);
        sum += f * l[x];
        others[tid][x] = f;
      }
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      if (x < p.cluster) { others[tid][x] = seen > 0.f ? others[tid][x] / sum : 0.f; }
    }
    weight[tid][0] = seen;
    if (rank == 0) { put_sums(p, g, tid, top - raise, sum, seen > 0.f); }
  }
  __syncthreads();
  // every block takes a part of the coordinates
  for (int e = rank * kThreads + tid; e < g.n_heads * p.dim; e += p.cluster * kThreads) {
    const int i = e / p.dim, c = e - i * p.dim;
    float v = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      if (x < p.cluster) { v += others[i][x] * *cluster.map_shared_rank(sums + i * kRow + c, x); }
    }
    put_out<T>(p, g, i, c, weight[i][0] > 0.f ? v : 0.f);
  }
  cluster.sync();  // the others may still read this block's memory
}

/// The softmax of a tile's scores s (R times 16 keys x 8 queries, as the first product leaves them), one group of eight queries:
/// scores become weights as the second product's operand, m and l go on. Returns whether m grew (in this thread's queries).
template <typename T, int R>
__device__ __forceinline__ bool soften(float (&s)[R][4], float scale, const bool (&see)[R][2], float (&m)[2], float (&l)[2], float (&alpha)[2],
                                       uint32_t (&hi)[R][2], uint32_t (&lo)[R][2])
{
  float base[2];
  bool grew = false;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r][c]     = see[r][0] ? s[r][c] * scale : -INFINITY;
      s[r][c + 2] = see[r][1] ? s[r][c + 2] * scale : -INFINITY;
      top         = fmaxf(top, fmaxf(s[r][c], s[r][c + 2]));
    }
    top      = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
    top      = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
    top      = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
    top      = fmaxf(top, m[c]);
    base[c]  = top == -INFINITY ? 0.f : top;
    alpha[c] = exp2_fast(m[c] - base[c]);
    grew     = grew || top > m[c];
    m[c]     = top;
    base[c] -= Half<T>::kRaise;
    l[c] *= alpha[c];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int c = 0; c < 4; ++c) { s[r][c] = exp2_fast(s[r][c] - base[c & 1]); }
    l[0] += s[r][0] + s[r][2];
    l[1] += s[r][1] + s[r][3];
    Half<T>::split(s[r][0], s[r][1], hi[r][0], lo[r][0]);
    Half<T>::split(s[r][2], s[r][3], hi[r][1], lo[r][1]);
    // from keys by lanes to queries by lanes
    hi[r][0] = transpose8x8(hi[r][0]), hi[r][1] = transpose8x8(hi[r][1]);
    lo[r][0] = transpose8x8(lo[r][0]), lo[r][1] = transpose8x8(lo[r][1]);
  }
  return grew;
}

/// The sum over the lanes that hold different keys of the same query.
__device__ __forceinline__ float sum_over_keys(float v)
{
  v += __shfl_xor_sync(~0u, v, 4);
  v += __shfl_xor_sync(~0u, v, 8);
  return v + __shfl_xor_sync(~0u, v, 16);
}

// Heads of up to 128 coordinates: operands come straight from global memory into the registers of the product that uses
// them. A product over coordinates may take them in any order, as long as keys and queries agree, so lane t of a
// key's four lanes takes 16 bytes in a row for two steps of the product; and the second product's rows, the
// coordinates of the result, may be any eight coordinates, so lane g of a value's eight lanes takes 16 bytes in a row for
// four products. What is left is to pair the values of neighbouring keys, one byte permutation per register.
// Against copies into shared memory and ldmatrix this takes 380 instructions per tile of 8 KB instead of 470.

/// N * 4 bytes that are read once (not by .nc: a block is there while the kernel in front still writes them).
template <int N>
__device__ __forceinline__ void read_once(uint32_t (&r)[N], const char* at)
{
  static_assert(N == 1 || N == 2 || N == 4, "");
  if constexpr (N == 4) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(at));
  } else if constexpr (N == 2) {
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(at));
  } else {
    asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(r[0]) : "l"(at));
  }
}

/// Narrow heads take 32 keys at a time: as many bytes in flight, and half the steps of the softmax. 16 rows of 16 384 keys of 8 heads
/// of 64: 116 us with 16 keys, 98 with 32; heads of 80: 131 and 128.
constexpr int kDoubleDim = 80;

/// A lane's share of a row's coordinates in blocks: 8 * E coordinates where every lane of eight (or 4 * E, of four) takes E.
template <int N64, int N32, int N16>
struct RowPart {
  uint32_t b64[N64 ? N64 : 1][4], b32[N32 ? N32 : 1][2], b16[N16 ? N16 : 1][1];
};

template <typename T, int D, int NT, bool PAD, int W>
__global__ void __launch_bounds__(W * 32, (NT == 1 ? 12 : 8) / W) attend_direct_kernel(const AttendParams p)
{
  constexpr int kK32 = D / 32, kK16 = D % 32 / 16;                  // keys: blocks of 32 and 16 coordinates
  constexpr int kV64 = D / 64, kV32 = D % 64 / 32, kV16 = D % 32 / 16;  // values: of 64, 32 and 16
  constexpr int kSteps = 2 * kK32 + kK16, kTiles = 4 * kV64 + 2 * kV32 + kV16;
  constexpr int R = D <= kDoubleDim ? 2 : 1, kKeys = 16 * R;  // keys of a tile
  extern __shared__ __align__(16) float sums[];  // [warps][8 NT][D + 4]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g8 = lane / 4, t4 = lane % 4;
  begin(p);

  for_segments<T, W>(p, [&](const Segment& g) {
    const char* keys   = static_cast<const char*>(p.keys) + g.kv * p.k_head * sizeof(T) + t4 * 16;
    const char* values = static_cast<const char*>(p.values) + g.kv * p.v_head * sizeof(T) + g8 * 16;
    const int i0 = g.i0, i1 = g.i1, begin = g.begin;
    const void* index  = g.index;
    const int tiles    = (i1 - i0 + kKeys - 1) / kKeys;
    const int n        = tiles > warp ? (tiles - warp + W - 1) / W : 0;

    // token lane % kKeys of tile j, its entry and its place
    auto token_of = [&](int j) { return i0 + (warp + j * W) * kKeys + lane % kKeys; };
    auto ask      = [&](int j) { return j < n && token_of(j) < i1 ? entry_of(p, begin, index, token_of(j)) : 0; };
    auto find     = [&](int j, int64_t entry) {
      return j < n && token_of(j) < i1 ? place_of(p, begin, token_of(j), entry) : Place{kNowhere, kNowhere};
    };
    int64_t entry0 = ask(0), entry = ask(1);

    // the queries, as the 8-column side of the first product; a lane takes the same coordinates of a query as of a key
    uint32_t qf[NT][kSteps][2];
    {
      const T* q = static_cast<const T*>(p.q) + int64_t(g.row) * p.q_row + g.head * p.q_head;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        const int i  = x * 8 + g8;
        const T* row = q + i * p.q_head;
        if (p.q_wide && i < g.n_heads) {
#pragma unroll
          for (int k = 0; k < kK32; ++k) {
            uint4 v{0, 0, 0, 0};
            if (!PAD || k * 32 + t4 * 8 < p.dim) { v = *reinterpret_cast<const uint4*>(row + k * 32 + t4 * 8); }
            qf[x][2 * k][0] = v.x, qf[x][2 * k][1] = v.y, qf[x][2 * k + 1][0] = v.z, qf[x][2 * k + 1][1] = v.w;
          }
          if constexpr (kK16 > 0) {
            const uint2 v = *reinterpret_cast<const uint2*>(row + kK32 * 32 + t4 * 4);
            qf[x][2 * kK32][0] = v.x, qf[x][2 * kK32][1] = v.y;
          }
        } else {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = k < 2 * kK32 ? k / 2 * 32 + t4 * 8 + k % 2 * 4 + h * 2 : kK32 * 32 + t4 * 4 + h * 2;
              uint32_t v  = 0;
              if (i < g.n_heads && (!PAD || c < p.dim)) {
                const auto a = *reinterpret_cast<const uint16_t*>(row + c), b = *reinterpret_cast<const uint16_t*>(row + c + 1);
                v            = a | (uint32_t(b) << 16);
              }
              qf[x][k][h] = v;
            }
          }
        }
      }
    }
    float o[NT][kTiles][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int d = 0; d < kTiles; ++d) { o[x][d][0] = o[x][d][1] = o[x][d][2] = o[x][d][3] = 0.f; }
      m[x][0] = m[x][1] = -INFINITY;
      l[x][0] = l[x][1] = 0.f;
    }

    // of every sixteen keys: keys g8 and g8 + 8, values of keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9
    uint32_t kr[2 * R][kK32 + kK16][4];
    RowPart<kV64, kV32, kV16> vr[4 * R];
    auto at_of = [&](uint32_t place) { return static_cast<uint64_t>(place == kNowhere ? 0 : place) << p.unit_shift; };
    auto load_keys = [&](const uint32_t (&place)[2 * R]) {
#pragma unroll
      for (int r = 0; r < 2 * R; ++r) {
        const char* at = keys + at_of(place[r]);
#pragma unroll
        for (int b = 0; b < kK32; ++b) {
          if (!PAD || b * 32 + t4 * 8 < p.dim) { read_once<4>(kr[r][b], at + b * 64); }
        }
        if constexpr (kK16 > 0) {
          uint32_t two[2];
          read_once<2>(two, at + kK32 * 64 - t4 * 8);
          kr[r][kK32][0] = two[0], kr[r][kK32][1] = two[1];
        }
      }
    };
    auto load_values = [&](const uint32_t (&place)[4 * R]) {
#pragma unroll
      for (int r = 0; r < 4 * R; ++r) {
        const char* at = values + at_of(place[r]);
#pragma unroll
        for (int b = 0; b < kV64; ++b) {
          if (!PAD || b * 64 + g8 * 8 < p.dim) { read_once<4>(vr[r].b64[b], at + b * 128); }
        }
        if constexpr (kV32 > 0) { read_once<2>(vr[r].b32[0], at + kV64 * 128 - g8 * 8); }
        if constexpr (kV16 > 0) { read_once<1>(vr[r].b16[0], at + kV64 * 128 + kV32 * 64 - g8 * 12); }
      }
    };
    auto keys_of = [&](const Place& x, uint32_t (&place)[2 * R]) {
#pragma unroll
      for (int r = 0; r < 2 * R; ++r) { place[r] = __shfl_sync(~0u, x.k, g8 + 8 * r); }
    };
    auto values_of = [&](const Place& x, uint32_t (&place)[4 * R]) {
#pragma unroll
      for (int r = 0; r < 4 * R; ++r) { place[r] = __shfl_sync(~0u, x.v, r / 4 * 16 + t4 * 2 + (r & 1) + (r & 2) * 4); }
    };
    // a register of two neighbouring keys' values at one coordinate
    auto pair = [](uint32_t a, uint32_t b, int odd) { return __byte_perm(a, b, odd ? 0x7632 : 0x5410); };

    if (PAD) {
      // what lies behind the last coordinate is never loaded, and must be a number
#pragma unroll
      for (int r = 0; r < 2 * R; ++r) {
#pragma unroll
        for (int b = 0; b < kK32; ++b) { kr[r][b][0] = kr[r][b][1] = kr[r][b][2] = kr[r][b][3] = 0; }
      }
#pragma unroll
      for (int r = 0; r < 4 * R; ++r) {
#pragma unroll
        for (int b = 0; b < kV64; ++b) { vr[r].b64[b][0] = vr[r].b64[b][1] = vr[r].b64[b][2] = vr[r].b64[b][3] = 0; }
      }
    }
    uint32_t kp[2 * R], vp[4 * R];
    bool any = false;
    if (n > 0) {
      const Place at = find(0, entry0);
      keys_of(at, kp);
      values_of(at, vp);
      load_keys(kp);
      load_values(vp);
    }
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      // where the next tile lies is worked out while this one's keys are on their way
      bool see[R][2], all = true;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        see[r][0] = kp[2 * r] != kNowhere, see[r][1] = kp[2 * r + 1] != kNowhere;
        any       = any || see[r][0] || see[r][1];
        all       = all && see[r][0] && see[r][1];
      }
      const Place at = find(j + 1, entry);
      entry          = ask(j + 2);
      keys_of(at, kp);
      float s[NT][R][4];
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int r = 0; r < R; ++r) { s[x][r][0] = s[x][r][1] = s[x][r][2] = s[x][r][3] = 0.f; }
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int b = k / 2, h = k % 2 * 2;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint32_t a[4] = {kr[2 * r][b][h], kr[2 * r + 1][b][h], kr[2 * r][b][h + 1], kr[2 * r + 1][b][h + 1]};
#pragma unroll
          for (int x = 0; x < NT; ++x) { Half<T>::mma(s[x][r], a, qf[x][k][0], qf[x][k][1]); }
        }
      }
      if (j + 1 < n) { load_keys(kp); }

      uint32_t hi[NT][R][2], lo[NT][R][2];
      float alpha[NT][2];
      bool grew = false;
#pragma unroll
      for (int x = 0; x < NT; ++x) { grew |= soften<T, R>(s[x], p.scale, see, m[x], l[x], alpha[x], hi[x], lo[x]); }
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
          for (int d = 0; d < kTiles; ++d) {
            o[x][d][0] *= alpha[x][0], o[x][d][1] *= alpha[x][1];
            o[x][d][2] *= alpha[x][0], o[x][d][3] *= alpha[x][1];
          }
        }
      }
      // every key of the tile is seen, or the values of those that are not become zeros
      if (!__all_sync(~0u, all)) {
#pragma unroll
        for (int r = 0; r < 4 * R; ++r) {
          if (vp[r] == kNowhere) {
#pragma unroll
            for (int b = 0; b < kV64; ++b) { vr[r].b64[b][0] = vr[r].b64[b][1] = vr[r].b64[b][2] = vr[r].b64[b][3] = 0; }
            vr[r].b32[0][0] = vr[r].b32[0][1] = vr[r].b16[0][0] = 0;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const auto* v = vr + 4 * r;
#pragma unroll
        for (int d = 0; d < kTiles; ++d) {
          uint32_t a[4];
          if (d < 4 * kV64) {
            const int b = d / 4, i = d % 4, h = i % 2;
            a[0] = pair(v[0].b64[b][i / 2], v[1].b64[b][i / 2], h), a[1] = pair(v[0].b64[b][i / 2 + 2], v[1].b64[b][i / 2 + 2], h);
            a[2] = pair(v[2].b64[b][i / 2], v[3].b64[b][i / 2], h), a[3] = pair(v[2].b64[b][i / 2 + 2], v[3].b64[b][i / 2 + 2], h);
          } else if (d < 4 * kV64 + 2 * kV32) {
            const int h = d % 2;
            a[0] = pair(v[0].b32[0][0], v[1].b32[0][0], h), a[1] = pair(v[0].b32[0][1], v[1].b32[0][1], h);
            a[2] = pair(v[2].b32[0][0], v[3].b32[0][0], h), a[3] = pair(v[2].b32[0][1], v[3].b32[0][1], h);
          } else {
            a[0] = pair(v[0].b16[0][0], v[1].b16[0][0], 0), a[1] = pair(v[0].b16[0][0], v[1].b16[0][0], 1);
            a[2] = pair(v[2].b16[0][0], v[3].b16[0][0], 0), a[3] = pair(v[2].b16[0][0], v[3].b16[0][0], 1);
          }
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            Half<T>::mma(o[x][d], a, hi[x][r][0], hi[x][r][1]);
            Half<T>::mma(o[x][d], a, lo[x][r][0], lo[x][r][1]);
          }
        }
      }
      values_of(at, vp);
      if (j + 1 < n) { load_values(vp); }
    }

    constexpr int kRow = D + 4, kPitch = 8 * NT * kRow;
    any = __any_sync(~0u, any);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* to = sums + warp * kPitch + (x * 8 + t4 * 2 + c) * kRow;
#pragma unroll
        for (int d = 0; d < kTiles; ++d) {
          // the coordinates of rows g8 and g8 + 8 of product d
          int at, step;
          if (d < 4 * kV64) {
            at = d / 4 * 64 + g8 * 8 + d % 4, step = 4;
          } else if (d < 4 * kV64 + 2 * kV32) {
            at = kV64 * 64 + g8 * 4 + d % 2, step = 2;
          } else {
            at = kV64 * 64 + kV32 * 32 + g8 * 2, step = 1;
          }
          to[at]        = o[x][d][c];
          to[at + step] = o[x][d][c + 2];
        }
        const float sum = sum_over_keys(l[x][c]);
        if (g8 == 0) { to[D] = m[x][c], to[D + 1] = sum, to[D + 2] = any ? 1.f : 0.f; }
      }
    }
    finish_segment<T, D, W>(p, g, sums, kPitch, Half<T>::kRaise);
  });
}

// Wider heads do not fit the registers that way: their tiles are copied into a ring in shared memory that belongs to a warp.
template <int D>  // the head dimension, padded to what the tiles are built for
struct HalfTile {
  static constexpr int kPitch = D * 2 + 16;  // bytes of a row in shared memory: eight rows start in eight different banks
  static constexpr int kBytes = kKeys * kPitch;
  static constexpr int kWarp  = kStages * 2 * kBytes;
};

template <typename T, int D, int NT, int W>
__global__ void __launch_bounds__(W * 32, 4 / W) attend_ring_kernel(const AttendParams p)
{
  using Tile = HalfTile<D>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g8 = lane / 4, t4 = lane % 4;
  unsigned char* ring = smem + warp * Tile::kWarp;
  const uint32_t ring_at = smem_of(ring);
  begin(p);
  if (p.dim < D) {
    // the columns behind the last coordinate are multiplied by zeros of the queries: they must hold numbers
    for (int i = lane * 16; i < Tile::kWarp; i += 32 * 16) { *reinterpret_cast<uint4*>(ring + i) = uint4{0, 0, 0, 0}; }
    __syncwarp();
  }

  for_segments<T, W>(p, [&](const Segment& g) {
    // the queries, as the 8-column side of the first product
    uint32_t qf[NT][D / 16][2];
    {
      const T* q = static_cast<const T*>(p.q) + int64_t(g.row) * p.q_row + g.head * p.q_head;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int i  = n * 8 + g8;
        const T* row = q + i * p.q_head;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = k * 16 + h * 8 + t4 * 2;
            uint32_t v  = 0;
            if (i < g.n_heads && c < p.dim) {
              const auto a = *reinterpret_cast<const uint16_t*>(row + c), b = *reinterpret_cast<const uint16_t*>(row + c + 1);
              v            = a | (uint32_t(b) << 16);
            }
            qf[n][k][h] = v;
          }
        }
      }
    }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d) { o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f; }
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

    const char* keys   = static_cast<const char*>(p.keys) + g.kv * p.k_head * sizeof(T);
    const char* values = static_cast<const char*>(p.values) + g.kv * p.v_head * sizeof(T);
    // tiles of this warp: warp, warp + W, ...
    const int i0 = g.i0, i1 = g.i1, begin = g.begin;
    const void* index = g.index;
    const int tiles   = (i1 - i0 + kKeys - 1) / kKeys;
    const int n     = tiles > warp ? (tiles - warp + W - 1) / W : 0;
    // token lane % 16 of tile j, its entry and its place
    auto token_of = [&](int j) { return i0 + (warp + j * W) * kKeys + lane % kKeys; };
    auto ask      = [&](int j) { return j < n && token_of(j) < i1 ? entry_of(p, begin, index, token_of(j)) : 0; };
    auto find     = [&](int j, int64_t entry) {
      return j < n && token_of(j) < i1 ? place_of(p, begin, token_of(j), entry) : Place{kNowhere, kNowhere};
    };
    uint32_t masks = 0;  // of the tiles in the ring: which keys are real, newest lowest
    uint32_t older = 0;
    auto copy = [&](int stage, const Place& at) {
      const uint32_t to = ring_at + stage * 2 * Tile::kBytes + lane * 16;
      const bool inside = lane * 8 < p.dim;
#pragma unroll
      for (int row = 0; row < kKeys; ++row) {
        const uint32_t ka = __shfl_sync(~0u, at.k, row), va = __shfl_sync(~0u, at.v, row);
        const bool ok     = ka != kNowhere;
        if (inside) {
          copy16(to + row * Tile::kPitch, keys + (ok ? static_cast<uint64_t>(ka) << p.unit_shift : 0) + lane * 16, ok);
          copy16(to + Tile::kBytes + row * Tile::kPitch, values + (ok ? static_cast<uint64_t>(va) << p.unit_shift : 0) + lane * 16, ok);
        }
      }
      older = masks >> 16;
      masks = (masks << 16) | (__ballot_sync(~0u, at.k != kNowhere) & 0xffffu);
    };
    bool any = false;
    static_assert(kStages == 3, "two tiles are copied ahead");
    {
      const int64_t first = ask(0), second = ask(1);
      copy(0, find(0, first));
      copy_commit();
      copy(1, find(1, second));
      copy_commit();
    }
    int64_t entry = ask(2);
    int stage     = 0;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      copy_wait<kStages - 2>();
      __syncwarp();
      copy(stage == 0 ? kStages - 1 : stage - 1, find(j + 2, entry));
      copy_commit();
      entry = ask(j + 3);
      const uint32_t mask = older & 0xffffu;  // kStages - 1 = 2 tiles were copied behind this one
      any                 = any || mask != 0;
      const uint32_t k_tile = ring_at + stage * 2 * Tile::kBytes, v_tile = k_tile + Tile::kBytes;
      stage = stage + 1 == kStages ? 0 : stage + 1;

      float s[NT][1][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) { s[i][0][0] = s[i][0][1] = s[i][0][2] = s[i][0][3] = 0.f; }
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t a[4];
        load_matrix(a, k_tile + (lane % 16) * Tile::kPitch + (k * 2 + lane / 16) * 16);
#pragma unroll
        for (int i = 0; i < NT; ++i) { Half<T>::mma(s[i][0], a, qf[i][k][0], qf[i][k][1]); }
      }
      const bool see[1][2] = {{(mask >> g8 & 1) != 0, (mask >> (g8 + 8) & 1) != 0}};
      uint32_t hi[NT][1][2], lo[NT][1][2];
      bool grew = false;
      float alpha[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) { grew |= soften<T, 1>(s[i], p.scale, see, m[i], l[i], alpha[i], hi[i], lo[i]); }
      if (__any_sync(~0u, grew)) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[i][d][0] *= alpha[i][0], o[i][d][1] *= alpha[i][1];
            o[i][d][2] *= alpha[i][0], o[i][d][3] *= alpha[i][1];
          }
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t a[4];
        load_matrix_t(a, v_tile + (lane % 8 + (lane / 16) * 8) * Tile::kPitch + (d * 2 + lane / 8 % 2) * 16);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          Half<T>::mma(o[i][d], a, hi[i][0][0], hi[i][0][1]);
          Half<T>::mma(o[i][d], a, lo[i][0][0], lo[i][0][1]);
        }
      }
    }
    copy_wait<0>();
    __syncwarp();

    // the warps' results meet in shared memory, each in its own ring
    constexpr int kRow = D + 4;
    auto* sums         = reinterpret_cast<float*>(ring);  // [8 NT][kRow]: output, m, l, any
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* to = sums + (i * 8 + t4 * 2 + c) * kRow;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          to[d * 16 + g8]     = o[i][d][c];
          to[d * 16 + g8 + 8] = o[i][d][c + 2];
        }
        const float sum = sum_over_keys(l[i][c]);
        if (g8 == 0) { to[D] = m[i][c], to[D + 1] = sum, to[D + 2] = any ? 1.f : 0.f; }
      }
    }
    finish_segment<T, D, W>(p, g, reinterpret_cast<float*>(smem), Tile::kWarp / 4, Half<T>::kRaise);
    if (p.dim < D) {
      for (int i = lane * 16; i < Tile::kWarp; i += 32 * 16) { *reinterpret_cast<uint4*>(ring + i) = uint4{0, 0, 0, 0}; }
      __syncwarp();
    }
  });
}

// ------------------------------------------------------------------------------------------------ float32
// No tensor core keeps float32's products, so this is fused multiply-adds, two at a time (fma.f32x2). Keys lie in registers like
// above, four lanes per key with 16 bytes in a row each; the queries come from shared memory, one read for both keys of a lane.
// The four lanes' parts of a score are added while the queries are dealt out to them. For the second product a lane owns four
// coordinates of every value, and the weights come from shared memory. 830 instructions per tile of 16 KB (8 queries, d = 128).
__device__ __forceinline__ void fma2(float2& d, float2 a, float2 b)
{
  auto& x = reinterpret_cast<unsigned long long&>(d);
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(x) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
}

template <int D, int Q, int W>
struct FloatTile {
  static constexpr int kPer    = D <= 128 ? 2 : 1;      // keys of a lane
  static constexpr int kKeys   = 8 * kPer;              // of a tile
  static constexpr int kChunks = D / 16;                // 16-byte parts of a key that a lane holds
  static constexpr int kRows   = D <= 64 ? 2 : 1;       // values that the warp reads at once
  static constexpr int kWide   = D <= 128 ? 1 : D / 128;  // 16-byte parts of a value that a lane holds
  static constexpr int kOwn    = Q >= 4 ? Q / 4 : 1;    // queries whose softmax a lane does
  static constexpr int kWeights = 2 * Q * kKeys + (Q < 4 ? 4 : Q);  // floats of a warp: weights, twice each for fma2, and factors
  static constexpr int kSums   = Q * (D + 4);           // of a warp: what it found
  static constexpr int kBytes  = 4 * (Q * D + W * (kWeights + kSums));
};

/// D: the head dimension, padded; Q: queries of a unit, padded to 1, 4 or 8.
template <int D, int Q, int W>
__global__ void __launch_bounds__(W * 32, 8 / W) attend_float_kernel(const AttendParams p)
{
  using Tile = FloatTile<D, Q, W>;
  constexpr int kPer = Tile::kPer, kKeys = Tile::kKeys, kChunks = Tile::kChunks, kRows = Tile::kRows, kWide = Tile::kWide, kOwn = Tile::kOwn;
  extern __shared__ __align__(16) float shared[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g8 = lane / 4, t4 = lane % 4;
  float* q_s     = shared;                                            // [Q][D]
  float* weights = q_s + Q * D + warp * Tile::kWeights;               // [Q][keys][2]
  float* factors = weights + 2 * Q * kKeys;                           // [Q]
  float* sums    = q_s + Q * D + W * Tile::kWeights;             // [warps][Q][D + 4]
  begin(p);

  for_segments<float, W>(p, [&](const Segment& g) {
    const char* keys   = static_cast<const char*>(p.keys) + g.kv * p.k_head * sizeof(float) + t4 * 16;
    const int column   = D <= 64 ? lane % 16 * 4 : lane * 4;  // the lane's first coordinate of a value
    const char* values = static_cast<const char*>(p.values) + g.kv * p.v_head * sizeof(float) + column * 4;
    const int i0 = g.i0, i1 = g.i1, begin = g.begin;
    const void* index  = g.index;
    const int tiles    = (i1 - i0 + kKeys - 1) / kKeys;
    const int n        = tiles > warp ? (tiles - warp + W - 1) / W : 0;
    auto token_of      = [&](int j) { return i0 + (warp + j * W) * kKeys + lane % kKeys; };
    auto ask           = [&](int j) { return j < n && token_of(j) < i1 ? entry_of(p, begin, index, token_of(j)) : 0; };
    auto find          = [&](int j, int64_t entry) {
      return j < n && token_of(j) < i1 ? place_of(p, begin, token_of(j), entry) : Place{kNowhere, kNowhere};
    };
    int64_t entry0 = ask(0), entry = ask(1);
    const float* q = static_cast<const float*>(p.q) + int64_t(g.row) * p.q_row + g.head * p.q_head;
    for (int i = threadIdx.x; i < Q * D; i += W * 32) {
      const int x = i / D, c = i % D;
      q_s[i] = x < g.n_heads && c < p.dim ? q[x * p.q_head + c] : 0.f;
    }
    __syncthreads();

    float4 kr[kPer][kChunks], vr[kKeys / kRows][kWide];
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) { kr[x][c] = float4{0.f, 0.f, 0.f, 0.f}; }
    }
#pragma unroll
    for (int x = 0; x < kKeys / kRows; ++x) {
#pragma unroll
      for (int c = 0; c < kWide; ++c) { vr[x][c] = float4{0.f, 0.f, 0.f, 0.f}; }
    }
    auto at_of     = [&](uint32_t place) { return static_cast<uint64_t>(place == kNowhere ? 0 : place) << p.unit_shift; };
    auto keys_of   = [&](const Place& at, uint32_t (&place)[kPer]) {
#pragma unroll
      for (int x = 0; x < kPer; ++x) { place[x] = __shfl_sync(~0u, at.k, g8 + 8 * x); }
    };
    auto load_keys = [&](const uint32_t (&place)[kPer]) {
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const char* from = keys + at_of(place[x]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (c * 16 + t4 * 4 < p.dim) { read_once<4>(reinterpret_cast<uint32_t(&)[4]>(kr[x][c]), from + c * 64); }
        }
      }
    };
    auto load_values = [&](const Place& at) {
#pragma unroll
      for (int x = 0; x < kKeys / kRows; ++x) {
        const char* from = values + at_of(__shfl_sync(~0u, at.v, x * kRows + (kRows == 2 ? lane / 16 : 0)));
#pragma unroll
        for (int c = 0; c < kWide; ++c) {
          if (column + c * 128 < p.dim) { read_once<4>(reinterpret_cast<uint32_t(&)[4]>(vr[x][c]), from + c * 512); }
        }
      }
    };

    float2 o[Q][kWide][2];
    float m[kOwn], l[kOwn];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
#pragma unroll
      for (int c = 0; c < kWide; ++c) { o[i][c][0] = o[i][c][1] = float2{0.f, 0.f}; }
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) { m[i] = -INFINITY, l[i] = 0.f; }
    bool any = false;
    Place now = find(0, entry0);
    uint32_t kp[kPer];
    keys_of(now, kp);
    if (n > 0) {
      load_keys(kp);
      load_values(now);
    }
    uint32_t seen = __ballot_sync(~0u, now.k != kNowhere);  // bit i: key i of the tile
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      // where the next tile lies is worked out while this one's keys are on their way
      const uint32_t mask = seen;
      now                 = find(j + 1, entry);
      entry               = ask(j + 2);
      seen                = __ballot_sync(~0u, now.k != kNowhere);
      keys_of(now, kp);
      float s[Q][kPer];
      {
        float2 sum[Q][kPer];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
#pragma unroll
          for (int x = 0; x < kPer; ++x) { sum[i][x] = float2{0.f, 0.f}; }
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
          for (int i = 0; i < Q; ++i) {
            const float4 w = *reinterpret_cast<const float4*>(q_s + i * D + c * 16 + t4 * 4);
#pragma unroll
            for (int x = 0; x < kPer; ++x) {
              fma2(sum[i][x], float2{w.x, w.y}, float2{kr[x][c].x, kr[x][c].y});
              fma2(sum[i][x], float2{w.z, w.w}, float2{kr[x][c].z, kr[x][c].w});
            }
          }
        }
#pragma unroll
        for (int i = 0; i < Q; ++i) {
#pragma unroll
          for (int x = 0; x < kPer; ++x) { s[i][x] = sum[i][x].x + sum[i][x].y; }
        }
      }
      any = any || (mask & ((1u << kKeys) - 1)) != 0;
      if (j + 1 < n) { load_keys(kp); }

      // the four lanes of a key add their parts; with four queries or more each ends with its own queries
      if constexpr (Q >= 4) {
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
#pragma unroll
          for (int i = 0; i < Q / 2; ++i) {
            const float mine = t4 & 2 ? s[i + Q / 2][x] : s[i][x], other = t4 & 2 ? s[i][x] : s[i + Q / 2][x];
            s[i][x] = mine + __shfl_xor_sync(~0u, other, 2);
          }
#pragma unroll
          for (int i = 0; i < Q / 4; ++i) {
            const float mine = t4 & 1 ? s[i + Q / 4][x] : s[i][x], other = t4 & 1 ? s[i][x] : s[i + Q / 4][x];
            s[i][x] = mine + __shfl_xor_sync(~0u, other, 1);
          }
        }
      } else {
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
          s[0][x] += __shfl_xor_sync(~0u, s[0][x], 2);
          s[0][x] += __shfl_xor_sync(~0u, s[0][x], 1);
        }
      }
      const int own = Q >= 4 ? t4 * kOwn : 0;  // the lane's first query
      bool grew     = false;
      float alpha[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
          s[i][x] = mask >> (g8 + 8 * x) & 1 ? s[i][x] * p.scale : -INFINITY;
          top     = fmaxf(top, s[i][x]);
        }
        top              = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
        top              = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
        top              = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
        top              = fmaxf(top, m[i]);
        const float base = top == -INFINITY ? 0.f : top;
        alpha[i]         = exp2_fast(m[i] - base);
        grew             = grew || top > m[i];
        m[i]             = top;
        l[i] *= alpha[i];
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
          const float w = exp2_fast(s[i][x] - base);
          l[i] += w;
          if (Q >= 4 || t4 == 0) { *reinterpret_cast<float2*>(weights + 2 * ((own + i) * kKeys + g8 + 8 * x)) = float2{w, w}; }
        }
      }
      if (__any_sync(~0u, grew)) {
        if (g8 == 0) {
#pragma unroll
          for (int i = 0; i < kOwn; ++i) { factors[own + i] = alpha[i]; }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          const float f = factors[i];
#pragma unroll
          for (int c = 0; c < kWide; ++c) {
            o[i][c][0].x *= f, o[i][c][0].y *= f;
            o[i][c][1].x *= f, o[i][c][1].y *= f;
          }
        }
      }
      __syncwarp();
      if ((mask & ((1u << kKeys) - 1)) != (1u << kKeys) - 1) {
#pragma unroll
        for (int x = 0; x < kKeys / kRows; ++x) {
          if (!(mask >> (x * kRows + (kRows == 2 ? lane / 16 : 0)) & 1)) {
#pragma unroll
            for (int c = 0; c < kWide; ++c) { vr[x][c] = float4{0.f, 0.f, 0.f, 0.f}; }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < Q; ++i) {
#pragma unroll
        for (int x = 0; x < kKeys / kRows; x += 2) {
          // the weights of two values of the lane
          float2 w[2];
          if constexpr (kRows == 1) {
            const float4 both = *reinterpret_cast<const float4*>(weights + 2 * (i * kKeys + x));
            w[0] = float2{both.x, both.y}, w[1] = float2{both.z, both.w};
          } else {
            w[0] = *reinterpret_cast<const float2*>(weights + 2 * (i * kKeys + x * 2 + lane / 16));
            w[1] = *reinterpret_cast<const float2*>(weights + 2 * (i * kKeys + x * 2 + 2 + lane / 16));
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int c = 0; c < kWide; ++c) {
              fma2(o[i][c][0], w[y], float2{vr[x + y][c].x, vr[x + y][c].y});
              fma2(o[i][c][1], w[y], float2{vr[x + y][c].z, vr[x + y][c].w});
            }
          }
        }
      }
      __syncwarp();
      if (j + 1 < n) { load_values(now); }
    }

    float* mine = sums + warp * Tile::kSums;
#pragma unroll
    for (int i = 0; i < Q; ++i) {
#pragma unroll
      for (int c = 0; c < kWide; ++c) {
        float4 v{o[i][c][0].x, o[i][c][0].y, o[i][c][1].x, o[i][c][1].y};
        if constexpr (kRows == 2) {
          v.x += __shfl_xor_sync(~0u, v.x, 16), v.y += __shfl_xor_sync(~0u, v.y, 16);
          v.z += __shfl_xor_sync(~0u, v.z, 16), v.w += __shfl_xor_sync(~0u, v.w, 16);
        }
        if (column + c * 128 < D) { *reinterpret_cast<float4*>(mine + i * (D + 4) + column + c * 128) = v; }
      }
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const float sum = sum_over_keys(l[i]);
      if (g8 == 0 && (Q >= 4 || t4 == 0)) {
        float* to = mine + ((Q >= 4 ? t4 * kOwn : 0) + i) * (D + 4) + D;
        to[0] = m[i], to[1] = sum, to[2] = any ? 1.f : 0.f;
      }
    }
    finish_segment<float, D, W>(p, g, sums, Tile::kSums, 0.f);
  });
}

// ------------------------------------------------------------------------------------------------ joining the shares
constexpr int kJoinThreads = 256;

// What is joined is numbered by units, or by the blocks that may have begun one. Partial results lie in the second slot of the
// block that began the unit and in the first slots of those of the shares behind it.
struct Joint {
  int32_t row, first;  // first: the share that begins the unit
  int32_t unit, beside;
  int32_t n;           // its shares; 0: there is nothing to join
};

/// Every thread of a joining kernel calls this: when it returns, the first kernel has ended and its results are there. (A kernel
/// that is launched ahead of another's end must not end before it.)
__device__ __forceinline__ Joint joint_of(const AttendParams& p, int32_t x)
{
  Joint j{0, 0, 0, 0, 0};
  int32_t id = 0;
  if (p.marks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (x >= p.joints) { return j; }
    j.n                = p.marks[2 * x + 1];
    const int32_t mark = p.marks[2 * x];
    id                 = p.by_unit ? x : mark;
    j.first            = p.by_unit ? mark : divide(x, p.abreast);
  } else {
    // One length, so every unit has the same steps. It is read ahead of the wait: every block of the first kernel has waited for all that
    // wrote it before it let this kernel in (begin() keeps that order, and this depends on it), so L2 has it; L1, which may keep what
    // an earlier kernel read, is passed by.
    const int32_t steps = x < p.joints ? steps_for(p, span_of<true>(p, 0).count) : 0;
    if (steps > 0) {
      const Split split(steps * p.n_rows * p.in_line, p.shares);
      const int32_t share = divide(x, p.abreast);
      int32_t at          = -1;  // the unit's number among those that lie behind one another
      if (p.by_unit) {
        id = x;
        at = p.abreast == 1 ? id : divide(id, p.units);
      } else if (share < split.shares) {
        at = divide(split.first_step(share + 1) - 1, steps);
        id = p.abreast == 1 ? at : at * p.units + (x - share * p.abreast);
      }
      if (at >= 0) {
        j.first         = split.share_of(at * steps + kLead);
        const int32_t n = split.share_of((at + 1) * steps - 1) - j.first + 1;
        if (n > 1 && (p.by_unit || j.first == share)) { j.n = n; }
      }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
  if (j.n > 0) {
    j.row    = divide(id, p.units);
    j.unit   = id - j.row * p.units;
    j.beside = p.abreast == 1 ? 0 : j.unit;
  }
  return j;
}

__device__ __forceinline__ const float* part_of(const AttendParams& p, const Joint& j, int x)
{
  return p.parts + int64_t(2 * ((j.first + x) * p.abreast + j.beside) + (x == 0 ? 1 : 0)) * p.part_floats;
}

/// Many units with few shares each: a warp joins one query of one of them, four shares at a time with a running maximum.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_many_kernel(const AttendParams p)
{
  const int32_t item = blockIdx.x * (kJoinThreads / 32) + threadIdx.x / 32, x = divide(item, p.per_unit);
  const int lane = threadIdx.x % 32, i = item - x * p.per_unit;
  const Joint j  = joint_of(p, x);
  if (j.n == 0) { return; }
  const Segment g = segment_of(p, j.row, Span{0, 0, 0}, j.unit);
  if (i >= g.n_heads) { return; }
  constexpr int kAhead = 4;
  float top = -INFINITY, sum = 0.f, seen = 0.f;
  float4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int y0 = 0; y0 < j.n; y0 += kAhead) {
    float4 s[kAhead], o[kAhead][2];
    float next = top;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      s[y] = float4{-INFINITY, 0.f, 0.f, 0.f};
      o[y][0] = o[y][1] = float4{0.f, 0.f, 0.f, 0.f};
      if (y0 + y < j.n) {
        const float* from = part_of(p, j, y0 + y);
        s[y]              = *reinterpret_cast<const float4*>(from + 4 * i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = lane * 4 + h * 128;
          if (c < p.dim) { o[y][h] = *reinterpret_cast<const float4*>(from + 4 * p.per_unit + i * p.dim + c); }
        }
      }
    }
#pragma unroll
    for (int y = 0; y < kAhead; ++y) { next = fmaxf(next, s[y].x); }
    const float base = next == -INFINITY ? 0.f : next, alpha = exp2_fast(top - base);
    top              = next;
    sum *= alpha;
#pragma unroll
    for (int h = 0; h < 2; ++h) { v[h].x *= alpha, v[h].y *= alpha, v[h].z *= alpha, v[h].w *= alpha; }
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const float f = exp2_fast(s[y].x - base);
      sum += f * s[y].y;
      seen += s[y].z;
#pragma unroll
      for (int h = 0; h < 2; ++h) { v[h].x += f * o[y][h].x, v[h].y += f * o[y][h].y, v[h].z += f * o[y][h].z, v[h].w += f * o[y][h].w; }
    }
  }
  T* out = static_cast<T*>(p.out) + int64_t(j.row) * p.o_row + (g.head + i) * p.o_head;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = lane * 4 + h * 128;
    if (c < p.dim) {
      const float r[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
      for (int y = 0; y < 4; ++y) { out[c + y] = Type<T>::down(seen > 0.f ? r[y] / sum : 0.f); }
    }
  }
  if (p.lse && lane == 0) { p.lse[int64_t(j.row) * p.n_heads + g.head + i] = seen > 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY; }
}

/// Few units with many shares each: block (x, i, z) joins query i of joint x, coordinates 4 * join_lanes * z on. Sums and outputs are
/// read at once.
constexpr int kJoinSums = 5;  // shares whose sums a thread reads

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttendParams p)
{
  extern __shared__ float weight[];  // [shares]
  __shared__ float red[3][kJoinThreads / 32];
  __shared__ float4 outs[kJoinThreads];
  const int i = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Joint j = joint_of(p, blockIdx.x);
  if (j.n == 0) { return; }
  const Segment g = segment_of(p, j.row, Span{0, 0, 0}, j.unit);
  if (i >= g.n_heads) { return; }
  const int n = j.n;
  auto part   = [&](int x) { return part_of(p, j, x); };
  const int lanes = p.join_lanes, groups = kJoinThreads / lanes, from_c = blockIdx.z * lanes * 4;
  const int c = from_c + threadIdx.x % lanes * 4, mine = threadIdx.x / lanes;

  // this thread's first outputs set out before the sums are known
  constexpr int kAhead = 8;
  float4 ahead[kAhead];
#pragma unroll
  for (int x = 0; x < kAhead; ++x) {
    if (c < p.dim && mine + x * groups < n) {
      ahead[x] = *reinterpret_cast<const float4*>(part(mine + x * groups) + 4 * p.per_unit + i * p.dim + c);
    }
  }
  // the largest m of all, then the weights, the sum and whether anything was seen
  float top = -INFINITY;
  float4 sums[kJoinSums];
#pragma unroll
  for (int y = 0; y < kJoinSums; ++y) {
    const int x = threadIdx.x + y * kJoinThreads;
    sums[y]     = x < n ? *reinterpret_cast<const float4*>(part(x) + 4 * i) : float4{-INFINITY, 0.f, 0.f, 0.f};
    top         = fmaxf(top, sums[y].x);
  }
  for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(~0u, top, o)); }
  if (lane == 0) { red[0][warp] = top; }
  __syncthreads();
  for (float r : red[0]) { top = fmaxf(top, r); }
  float sum = 0.f, seen = 0.f;
#pragma unroll
  for (int y = 0; y < kJoinSums; ++y) {
    const int x   = threadIdx.x + y * kJoinThreads;
    const float f = top == -INFINITY ? 1.f : exp2_fast(sums[y].x - top);
    if (x < n) { weight[x] = f; }
    sum += f * sums[y].y;
    seen += sums[y].z;
  }
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, o);
    seen += __shfl_xor_sync(~0u, seen, o);
  }
  if (lane == 0) { red[1][warp] = sum, red[2][warp] = seen; }
  __syncthreads();
  sum = seen = 0.f;
  for (int x = 0; x < kJoinThreads / 32; ++x) { sum += red[1][x], seen += red[2][x]; }
  float4 v{0.f, 0.f, 0.f, 0.f};
  auto add = [&](float f, const float4& o) { v.x += f * o.x, v.y += f * o.y, v.z += f * o.z, v.w += f * o.w; };
  if (c < p.dim) {
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      if (mine + x * groups < n) { add(weight[mine + x * groups], ahead[x]); }
    }
#pragma unroll 8
    for (int x = mine + kAhead * groups; x < n; x += groups) {
      add(weight[x], *reinterpret_cast<const float4*>(part(x) + 4 * p.per_unit + i * p.dim + c));
    }
  }
  outs[threadIdx.x] = v;
  __syncthreads();
  for (int x = threadIdx.x; x < min(lanes * 4, p.dim - from_c); x += kJoinThreads) {
    float r = 0.f;
    for (int y = 0; y < groups; ++y) { r += reinterpret_cast<const float*>(outs + y * lanes)[x]; }
    (static_cast<T*>(p.out) + int64_t(g.row) * p.o_row + (g.head + i) * p.o_head)[from_c + x] = Type<T>::down(seen > 0.f ? r / sum : 0.f);
  }
  if (p.lse && threadIdx.x == 0 && blockIdx.z == 0) {
    p.lse[int64_t(g.row) * p.n_heads + g.head + i] = seen > 0.f ? (top + log2f(sum)) * kLn2 : -INFINITY;
  }
}

// ------------------------------------------------------------------------------------------------ launch
template <typename Kernel>
void launch(Kernel kernel, int warps, int smem, const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  // (40 KB: what needs no opt-in, with room for static shared memory)
  if (smem > 40 * 1024) { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); }
  cudaLaunchConfig_t c{};
  c.gridDim          = dim3(static_cast<unsigned>(blocks));
  c.blockDim         = dim3(warps * 32);
  c.dynamicSmemBytes = smem;
  c.stream           = s;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id               = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  c.attrs    = at;
  c.numAttrs = p.cluster <= 1 ? 1 : 2;
  cudaLaunchKernelEx(&c, kernel, p);
}

template <typename T, int D, bool PAD, int W>
void launch_direct(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  constexpr int kSums = W * 8 * (D + 4) * 4;
  if (p.per_unit <= 8) {
    launch(attend_direct_kernel<T, D, 1, PAD, W>, W, kSums, p, blocks, s);
  } else {
    launch(attend_direct_kernel<T, D, 2, PAD, W>, W, 2 * kSums, p, blocks, s);
  }
}
template <typename T, int D, bool PAD>
void launch_direct(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  p.warps == 4 ? launch_direct<T, D, PAD, 4>(p, blocks, s) : launch_direct<T, D, PAD, 2>(p, blocks, s);
}

template <typename T, int D, int W>
void launch_ring(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  if (p.per_unit <= 8) {
    launch(attend_ring_kernel<T, D, 1, W>, W, W * HalfTile<D>::kWarp, p, blocks, s);
  } else {
    launch(attend_ring_kernel<T, D, 2, W>, W, W * HalfTile<D>::kWarp, p, blocks, s);
  }
}
template <typename T, int D>
void launch_ring(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  p.warps == 4 ? launch_ring<T, D, 4>(p, blocks, s) : launch_ring<T, D, 2>(p, blocks, s);
}

template <typename T>
void launch_half(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  switch (p.dim) {
    case 64: return launch_direct<T, 64, false>(p, blocks, s);
    case 80: return launch_direct<T, 80, false>(p, blocks, s);
    case 96: return launch_direct<T, 96, false>(p, blocks, s);
    case 128: return launch_direct<T, 128, false>(p, blocks, s);
  }
  if (p.dim < 64) {
    launch_direct<T, 64, true>(p, blocks, s);
  } else if (p.dim < 128) {
    launch_direct<T, 128, true>(p, blocks, s);
  } else if (p.dim <= 192) {
    launch_ring<T, 192>(p, blocks, s);
  } else {
    launch_ring<T, 256>(p, blocks, s);
  }
}

template <int D, int W>
void launch_float(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  if (p.per_unit == 1) {
    launch(attend_float_kernel<D, 1, W>, W, FloatTile<D, 1, W>::kBytes, p, blocks, s);
  } else if (p.per_unit <= 4) {
    launch(attend_float_kernel<D, 4, W>, W, FloatTile<D, 4, W>::kBytes, p, blocks, s);
  } else {
    launch(attend_float_kernel<D, 8, W>, W, FloatTile<D, 8, W>::kBytes, p, blocks, s);
  }
}
template <int D>
void launch_float(const AttendParams& p, int64_t blocks, cudaStream_t s)
{
  p.warps == 4 ? launch_float<D, 4>(p, blocks, s) : launch_float<D, 1>(p, blocks, s);
}

template <typename T>
void launch_join(const AttendParams& p, cudaStream_t s)
{
  cudaLaunchConfig_t c{};
  c.blockDim = dim3(kJoinThreads);
  c.stream   = s;
  if (p.join_lanes == 0) {
    c.gridDim = dim3(static_cast<unsigned>((p.joints * p.per_unit * 32 + kJoinThreads - 1) / kJoinThreads));
  } else {
    c.gridDim          = dim3(static_cast<unsigned>(p.joints), static_cast<unsigned>(p.per_unit),
                              static_cast<unsigned>((p.dim + p.join_lanes * 4 - 1) / (p.join_lanes * 4)));
    c.dynamicSmemBytes = sizeof(float) * static_cast<size_t>(p.shares);
  }
  cudaLaunchAttribute early{};
  early.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  c.attrs                                          = &early;
  c.numAttrs                                       = 1;
  cudaLaunchKernelEx(&c, p.join_lanes == 0 ? join_many_kernel<T> : join_kernel<T>, p);
}

}  // namespace
}  // namespace certex_b200
