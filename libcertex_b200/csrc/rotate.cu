// Rotation of queries and keys by their positions, alone (certexB200Rotate) and on the way into a paged cache
// (certexB200PagedAppend).
//
// A pair (x0, x1) of a head's first r coordinates is turned by the angle a = position * w_i:
//   y0 = m (x0 cos a - x1 sin a),  y1 = m (x1 cos a + x0 sin a),
// pairs (2i, 2i + 1) when interleaved, (i, i + r / 2) otherwise. The inverse turns by -a, which is also the gradient.
//
// Angles. cos and sin see the angle modulo one turn only, so w_i is kept as a fraction of a turn in units of 2^-64 and
// position * w_i is the wrapping 64-bit product: the reduction to one turn is exact at every position, with an error of
// position * 2^-65 turns from the rounding of w_i. For float32 outputs the nearest quarter of a turn comes off in whole numbers as well:
// what is rounded to float32 is an eighth of a turn at most, and Taylor's series to the ninth and tenth power (what they leave out is
// 1.8e-9 and 1.2e-10 there) gives sines and cosines to a few units of their own last place, small ones too. (With half a turn
// rounded to float32 they were off by up to 1.1e-7, now by 5e-8; 200 000 rows of one head of 256 take 92 us instead of 95.)
// 16-bit outputs take the upper 32 bits as an angle in [-1/2, 1/2) turns and the hardware's sine and cosine of it, whose absolute error of
// 2^-20.9 on [-pi, pi] lies far below half a step of their types (2^-12 of the larger coordinate of a pair and more): the series instead costs
// a row of one head 30 % (100 000 rows of 128: 17.6 us for 13.3).
//
// One kernel for both. It moves bytes: everything is read once and written once, and what bounds it is HBM (32 768 rows of 32
// bfloat16 heads of 128 in 84 us, 6.4 TB/s; 16 384 rows appended with 32 query heads and 8 KV heads in 66, 6.1 TB/s) or the launch
// (a decoding step, 2 us). A thread owns one "unit" of a head: two vectors of 16 bytes that hold V whole pairs
// (neighbouring vectors when interleaved, a vector of each half otherwise), so that a pair never crosses threads and the
// call may be in place. It goes through up to eight heads with the same V sines and cosines: they depend on the row and the
// pair alone; where that is one head, a thread takes a key and its value.
#include "paged.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace certex_b200 {
namespace {

/// Two neighbouring 16-bit values as floats and back, and single ones.
__device__ __forceinline__ float2 up2(uint32_t w, __half)
{
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 up2(uint32_t w, __nv_bfloat16) { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
__device__ __forceinline__ uint32_t down2(float x, float y, __half)
{
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t down2(float x, float y, __nv_bfloat16)
{
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(__half v) { return __half2float(v); }
__device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float down(float v, float) { return v; }
__device__ __forceinline__ __half down(float v, __half) { return __float2half_rn(v); }
__device__ __forceinline__ __nv_bfloat16 down(float v, __nv_bfloat16) { return __float2bfloat16_rn(v); }

/// V elements that move as one access (V * sizeof(T) is 16, or V is 1).
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T e[V];
};

/// Heads that are treated alike: [rows, heads, dim] from `src` to `dst`, or to the cache (pages != null).
template <typename T>
struct Section {
  const T* src;
  int64_t src_row, src_head;
  T* dst;
  int64_t dst_row, dst_head;       // into rows; into pages: dst_row is the page's stride
  int64_t dst_token;               // into pages: a token's stride
  int32_t heads;
  int32_t chunks;                  // ceil(heads / heads of a thread)
  bool turn, paged;
};


template <typename T>
struct TurnArgs {
  Section<T> sec[3];
  int32_t n_sec;  // sections that have threads of their own; the values after them, where a thread takes a key and its value
  const uint64_t* turns;
  int32_t rotary_dim, dim;
  float magnitude;
  bool inverse;
  const void* positions;
  bool positions_64;
  int64_t n_rows;
  // pages
  certexB200PageTable_t table;
  int64_t n_pages, page_size;
  int32_t* fault;
};

/// a / b for a >= 0, in 32 bits where they will do.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b)
{
  return (a | b) >> 31 ? a / b : int64_t(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}

/// The sine and cosine of `turn` (in units of 2^-64 of a turn).
template <bool EXACT>
__device__ __forceinline__ void turn_sincos(uint64_t turn, float& s, float& c)
{
  if (EXACT) {
    const auto low      = static_cast<int32_t>(turn);
    const uint32_t high = static_cast<uint32_t>(turn >> 32) + (static_cast<uint32_t>(low) >> 31);  // turn = high 2^32 + low
    // four times what is left of the angle, in units of 2^-32 of a turn: the upper two bits of high are whole quarters
    const float rest = fmaf(static_cast<float>(low), 0x1p-30f, static_cast<float>(static_cast<int32_t>(high << 2)));
    // sin(pi t) and cos(pi t) for |t| <= 1/4 with coefficients pi^n / n!; pi itself in two parts
    const float t = rest * 0x1p-33f, t2 = t * t;
    float sine   = fmaf(8.214588661e-02f, t2, -5.992645293e-01f);
    sine         = fmaf(fmaf(sine, t2, 2.550164040e+00f), t2, -5.167712780e+00f);
    sine         = fmaf(t, 3.1415927410125732f, t * fmaf(t2, sine, -8.742278013e-08f));
    float cosine = fmaf(-2.580689139e-02f, t2, 2.353306304e-01f);
    cosine       = fmaf(fmaf(fmaf(cosine, t2, -1.335262769e+00f), t2, 4.058712126e+00f), t2, -4.934802201e+00f);
    cosine       = fmaf(cosine, t2, 1.f);
    // a quarter on, the sine is the cosine and the cosine minus the sine
    const uint32_t quarters = high + (1u << 29);
    const bool odd          = (quarters >> 30 & 1) != 0;
    s = __uint_as_float(__float_as_uint(odd ? cosine : sine) ^ (quarters & 0x80000000u));
    c = __uint_as_float(__float_as_uint(odd ? sine : cosine) ^ ((quarters + (1u << 30)) & 0x80000000u));
  } else {
    const float r = static_cast<float>(static_cast<int32_t>(turn >> 32)) * (3.14159265358979f * 0x1p-31f);
    s             = __sinf(r);
    c             = __cosf(r);
  }
}

/// The V pairs of a unit's vectors x and y turned by (c, s): pair i is (x[i], y[i]), or when interleaved the elements 2i and
/// 2i + 1 of both vectors in a row.
template <typename T, int V, bool INTERLEAVED>
__device__ __forceinline__ void turn_unit(Pack<T, V>& x, Pack<T, V>& y, const float (&c)[V], const float (&s)[V])
{
  if constexpr (sizeof(T) == 2 && V > 1) {
    auto* xw = reinterpret_cast<uint32_t*>(&x);
    auto* yw = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 u = up2(xw[i], T{}), w = up2(yw[i], T{});
      if constexpr (INTERLEAVED) {
        constexpr int H = V / 2;
        xw[i] = down2(u.x * c[i] - u.y * s[i], u.y * c[i] + u.x * s[i], T{});
        yw[i] = down2(w.x * c[H + i] - w.y * s[H + i], w.y * c[H + i] + w.x * s[H + i], T{});
      } else {
        xw[i] = down2(u.x * c[2 * i] - w.x * s[2 * i], u.y * c[2 * i + 1] - w.y * s[2 * i + 1], T{});
        yw[i] = down2(w.x * c[2 * i] + u.x * s[2 * i], w.y * c[2 * i + 1] + u.y * s[2 * i + 1], T{});
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      T& e0 = INTERLEAVED ? (2 * i < V ? x.e[(2 * i) % V] : y.e[(2 * i) % V]) : x.e[i];
      T& e1 = INTERLEAVED ? (2 * i + 1 < V ? x.e[(2 * i + 1) % V] : y.e[(2 * i + 1) % V]) : y.e[i];
      const float u = up(e0), w = up(e1);
      e0 = down(u * c[i] - w * s[i], T{});
      e1 = down(w * c[i] + u * s[i], T{});
    }
  }
}

// Four blocks of 256 threads on an SM with two heads' 64 bytes in flight per thread: 64 KB in flight. With four heads in flight
// in 159 registers there was room for one block, and turning 32 768 rows of 32 heads took 143 us.
template <typename T, int V, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(256, 4) turn_rows_kernel(const TurnArgs<T> a)
{
  constexpr bool kExact = sizeof(T) == 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the blocks are there before the kernel in front of them has ended
  const int units       = a.dim / (2 * V);  // of a head
  int chunks            = 0;
  for (int i = 0; i < a.n_sec; ++i) { chunks += a.sec[i].chunks; }
  const int64_t item = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int per      = chunks * units;
  const int64_t row  = item >> 31 ? item / per : static_cast<uint32_t>(item) / static_cast<uint32_t>(per);
  if (row >= a.n_rows) { return; }
  const int in_row = static_cast<int>(item - row * per);
  int chunk        = in_row / units;
  const int unit   = in_row - chunk * units;
  int which        = 0;
  while (chunk >= a.sec[which].chunks) { chunk -= a.sec[which++].chunks; }
  const Section<T> sec = which == 0 ? a.sec[0] : which == 1 ? a.sec[1] : a.sec[2];

  const int64_t pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[row] : static_cast<const int32_t*>(a.positions)[row];

  // where the unit's two vectors lie, and its first pair
  const int turned = a.rotary_dim / (2 * V);  // units that are turned
  const bool turn  = sec.turn && unit < turned;
  int lo = unit * 2 * V, hi = lo + V;
  if (!INTERLEAVED && unit < turned) {
    lo = unit * V;
    hi = lo + a.rotary_dim / 2;
  }
  using P           = Pack<T, V>;
  const int first   = chunk * HEADS;
  const T* from     = sec.src + row * sec.src_row + int64_t(first) * sec.src_head;
  const int n       = min(HEADS, sec.heads - first);
  constexpr int kAt = HEADS < 2 ? HEADS : 2;  // heads whose loads are in flight together
  P x[kAt], y[kAt];
  auto load = [&](int h) {
#pragma unroll
    for (int j = 0; j < kAt; ++j) {
      if (h + j < n) {
        x[j] = *reinterpret_cast<const P*>(from + j * sec.src_head + lo);
        y[j] = *reinterpret_cast<const P*>(from + j * sec.src_head + hi);
      }
    }
    from += kAt * sec.src_head;
  };
  load(0);  // on their way while the page is looked up
  const Section<T>& values = a.sec[HEADS == 1 ? a.n_sec : 0];
  P x2, y2;
  if (HEADS == 1 && sec.paged) {
    const T* from2 = values.src + row * values.src_row + int64_t(first) * values.src_head;
    x2             = *reinterpret_cast<const P*>(from2 + lo);
    y2             = *reinterpret_cast<const P*>(from2 + hi);
  }

  int64_t to = row * sec.dst_row;
  if (sec.paged) {
    if (pos < 0) { return; }  // a row that holds no token
    const int64_t b = a.table.row_to_sequence ? a.table.row_to_sequence[row] : row;
    const int64_t p = divide(pos, a.page_size);
    int64_t page    = -1;
    if (b >= 0 && b < a.table.n_sequences && p < a.table.pages_per_sequence) { page = a.table.pages[b * a.table.row_stride + p]; }
    if (page < 0 || page >= a.n_pages) {
      if (a.fault) { *a.fault = 1; }
      return;
    }
    to = page * sec.dst_row + (pos - p * a.page_size) * sec.dst_token;
    if (HEADS == 1) {
      T* dst2 = values.dst + page * values.dst_row + (pos - p * a.page_size) * values.dst_token + int64_t(first) * values.dst_head;
      *reinterpret_cast<P*>(dst2 + lo) = x2;
      *reinterpret_cast<P*>(dst2 + hi) = y2;
    }
  }
  T* dst = sec.dst + to + int64_t(first) * sec.dst_head;
  float c[V], s[V];
  if (turn) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      turn_sincos<kExact>(static_cast<uint64_t>(pos) * a.turns[unit * V + i], s[i], c[i]);
      c[i] *= a.magnitude;
      s[i] *= a.inverse ? -a.magnitude : a.magnitude;
    }
  }
#pragma unroll 1
  for (int h = 0; h < n; h += kAt) {
    if (h > 0) { load(h); }
#pragma unroll
    for (int j = 0; j < kAt; ++j) {
      if (h + j < n) {
        if (turn) { turn_unit<T, V, INTERLEAVED>(x[j], y[j], c, s); }
        *reinterpret_cast<P*>(dst + j * sec.dst_head + lo) = x[j];
        *reinterpret_cast<P*>(dst + j * sec.dst_head + hi) = y[j];
      }
    }
    dst += kAt * sec.dst_head;
  }
}

template <typename T, int V, int HEADS>
void run(TurnArgs<T>& a, bool interleaved, cudaStream_t s)
{
  int64_t chunks = 0;
  for (int i = 0; i < a.n_sec; ++i) {
    a.sec[i].chunks = (a.sec[i].heads + HEADS - 1) / HEADS;
    chunks += a.sec[i].chunks;
  }
  const int64_t items = a.n_rows * chunks * (a.dim / (2 * V));
  const int threads   = 256;
  const auto grid     = static_cast<unsigned>((items + threads - 1) / threads);
  cudaLaunchConfig_t c{};
  c.gridDim  = dim3(grid);
  c.blockDim = dim3(threads);
  c.stream   = s;
  cudaLaunchAttribute early{};
  early.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  c.attrs                                          = &early;
  c.numAttrs                                       = 1;
  cudaLaunchKernelEx(&c, interleaved ? turn_rows_kernel<T, V, true, HEADS> : turn_rows_kernel<T, V, false, HEADS>, a);
}

template <typename T, int V>
void run(TurnArgs<T>& a, bool interleaved, int sm_count, cudaStream_t s)
{
  int64_t heads = 0;
  for (int i = 0; i < a.n_sec; ++i) { heads += a.sec[i].heads; }
  // As many heads of a thread share its sines and cosines, and the row's page, as leave two blocks on every SM, and as the
  // sections come out even with: turning 4099 rows of 32 float32 heads takes 34 us with one head a thread and 21 with eight,
  // 16 384 rows of 12 bfloat16 heads 18 us with eight and 15 with four.
  const int64_t items = a.n_rows * heads * (a.dim / (2 * V)), wave = int64_t(sm_count) * 2 * 256;
  auto fits           = [&](int n) {
    bool even = items >= n * wave;
    for (int i = 0; i < a.n_sec; ++i) { even = even && (a.sec[i].heads + n - 1) / n * n * 4 <= a.sec[i].heads * 5; }
    return even;
  };
  if (fits(8)) {
    run<T, V, 8>(a, interleaved, s);
  } else if (fits(4)) {
    run<T, V, 4>(a, interleaved, s);
  } else if (fits(2)) {
    run<T, V, 2>(a, interleaved, s);
  } else {
    // few heads or few rows: a thread takes a key and its value, with one look at the table (keys and values of 73 324 rows of one
    // head 28 us apart and 21 together)
    if (a.sec[a.n_sec - 1].paged) { --a.n_sec; }
    run<T, V, 1>(a, interleaved, s);
  }
}

/// Whether every vector of these rows lies on its 16 bytes.
template <typename T>
bool aligned(const Section<T>& s)
{
  constexpr int V = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(s.src) % 16 == 0 && reinterpret_cast<uintptr_t>(s.dst) % 16 == 0 && s.src_row % V == 0 &&
         s.src_head % V == 0 && s.dst_row % V == 0 && s.dst_head % V == 0 && s.dst_token % V == 0;
}

template <typename T>
void turn(TurnArgs<T>& a, bool interleaved, int sm_count, cudaStream_t s)
{
  constexpr int V = 16 / sizeof(T);
  bool wide       = a.dim % (2 * V) == 0 && a.rotary_dim % (2 * V) == 0;
  for (int i = 0; i < a.n_sec; ++i) { wide = wide && aligned(a.sec[i]); }
  wide ? run<T, V>(a, interleaved, sm_count, s) : run<T, 1>(a, interleaved, sm_count, s);
}

template <typename T>
Section<T> section(const certexB200Rows_t& x, const certexB200Rows_t& y, int64_t heads, bool turned)
{
  return {static_cast<const T*>(x.data), x.row_stride, x.head_stride, static_cast<T*>(y.data), y.row_stride, y.head_stride, 0,
          static_cast<int32_t>(heads), 0, turned, false};
}

template <typename T>
TurnArgs<T> turn_args(const certexB200Rotary_t* plan, int64_t dim, const void* positions, bool positions_64, int64_t n_rows)
{
  TurnArgs<T> a{};
  a.turns        = plan ? plan->turns : nullptr;
  a.rotary_dim   = plan ? static_cast<int32_t>(plan->rotary_dim) : 0;
  a.magnitude    = plan ? static_cast<float>(plan->magnitude) : 1.0f;
  a.dim          = static_cast<int32_t>(dim);
  a.positions    = positions;
  a.positions_64 = positions_64;
  a.n_rows       = n_rows;
  a.page_size    = 1;
  return a;
}

template <typename F>
void by_type(int dtype, F&& f)
{
  if (dtype == kPagedF32) {
    f(float{});
  } else if (dtype == kPagedF16) {
    f(__half{});
  } else {
    f(__nv_bfloat16{});
  }
}

}  // namespace

void launch_rotate(const certexB200Rotary_t& plan, const certexB200Rows_t& x, const certexB200Rows_t& y, int64_t n_rows,
                   int64_t n_heads, int64_t head_dim, int dtype, const void* positions, bool positions_64, bool inverse,
                   int sm_count, cudaStream_t s)
{
  by_type(dtype, [&](auto t) {
    using T         = decltype(t);
    TurnArgs<T> a   = turn_args<T>(&plan, head_dim, positions, positions_64, n_rows);
    a.inverse       = inverse;
    a.sec[a.n_sec++] = section<T>(x, y, n_heads, true);
    turn(a, plan.interleaved != 0, sm_count, s);
  });
}

void launch_paged_append(const certexB200PagedCache_t& cache, const certexB200Rotary_t* plan, const certexB200PageTable_t& table,
                         const certexB200Rows_t& k, const certexB200Rows_t& v, const certexB200Rows_t& q,
                         const certexB200Rows_t& q_out, int64_t n_rows, int64_t n_q_heads, const void* positions,
                         bool positions_64, int sm_count, cudaStream_t s)
{
  by_type(static_cast<int>(cache.dtype), [&](auto t) {
    using T       = decltype(t);
    TurnArgs<T> a = turn_args<T>(plan, cache.head_dim, positions, positions_64, n_rows);
    a.table       = table;
    a.n_pages     = cache.n_pages;
    a.page_size   = cache.page_size;
    a.fault       = cache.fault;
    if (n_q_heads > 0) { a.sec[a.n_sec++] = section<T>(q, q_out, n_q_heads, true); }
    auto pages = [&](const certexB200Rows_t& from, void* to, const int64_t* strides, bool turned) {
      Section<T> x = section<T>(from, {to, strides[0], strides[2]}, cache.n_kv_heads, turned);
      x.dst_token  = strides[1];
      x.paged      = true;
      return x;
    };
    a.sec[a.n_sec++] = pages(k, cache.keys, cache.key_strides, plan != nullptr);
    a.sec[a.n_sec++] = pages(v, cache.values, cache.value_strides, false);
    turn(a, plan && plan->interleaved != 0, sm_count, s);
  });
}

}  // namespace certex_b200
