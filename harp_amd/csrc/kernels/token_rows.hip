// Rows of logits: log probabilities of given tokens with entropy and best alternatives, and the
// distillation loss against a teacher's top logits, with their gradients.
//
// With c the scale (1 / temperature), m a row's largest logit and S = sum_i exp(c (z_i - m)):
//   log p_i = c (z_i - m) - log S          H = log S - sum_i c (z_i - m) exp(c (z_i - m)) / S
// Both terms of H are >= 0, so a peaked row's small entropy is not a difference of large numbers.
// The pair (m, log S) is what the gradients read: c m + log S in one f32 would lose log S in rows
// whose logits are large, rows of the type's lowest value among them.
#include "elements.hpp"

namespace eh {
namespace {

constexpr float kLowest = -3.402823466e+38f;
constexpr int kCandidates = 256;          // elements at or above the selection's threshold that LDS holds

// A segment of a row as items of N elements that start at 16-byte boundaries, whatever the row's own
// start: item i has elements [N i - skew, N i - skew + N) of the segment, the first and the last item
// perhaps fewer.  (Vectors from an odd address cost a sixth of a reading pass's rate in 16-bit types.)
template <int DT> struct Segment {
  static constexpr int N = Elem<DT>::N;
  typedef typename Elem<DT>::T T;
  const T* p;
  int n, skew;
  __device__ Segment(const T* p_, int n_) : p(p_), n(n_), skew(static_cast<int>(reinterpret_cast<uintptr_t>(p_) / sizeof(T) % N)) {}
  __device__ int items() const { return (n + skew + N - 1) / N; }
  __device__ int full() const { return (n + skew) / N; }              // items before this one reach to their end
  __device__ int place(int i, int j) const { return i * N + j - skew; }
  __device__ u32x4 vector(int i) const { return *reinterpret_cast<const u32x4*>(p + (static_cast<int64_t>(i) * N - skew)); }
  // any item; what is not of the segment is -infinity
  __device__ void load(int i, float* z) const {
    if (i * N >= skew && i < full()) {
      Elem<DT>::unpack(vector(i), z);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int at = place(i, j);
        z[j] = at >= 0 && at < n ? Elem<DT>::get(p[at]) : -INFINITY;
      }
    }
  }
};

// ---- one pass over a row: running maximum, sum of exponentials, sum of their arguments -------------

struct RowSums {
  float largest = -INFINITY;     // over the elements themselves (NaN left out)
  float m = kLowest;             // what the sums are relative to: finite, so that m - m is 0 in a row of -infinity
  float s = 0.f;                 // sum exp2(c2 (z - m)); NaN if an element is NaN or +infinity
  float t = 0.f;                 // sum c2 (z - m) exp2(c2 (z - m))
};

template <bool ENT> __device__ inline void rebase(RowSums& a, float m, float c2) {
  const float d = (a.m - m) * c2, r = exp2_hw(d);
  if (ENT) a.t = (a.t + a.s * fmaxf(d, -1e20f)) * r;      // d is -infinity where nothing was summed yet
  a.s *= r;
  a.m = m;
}

template <int COUNT, bool ENT> __device__ inline void add_elements(RowSums& a, const float* z, float c2) {
  float b = max3(z[0], z[1], z[2]);
#pragma unroll
  for (int i = 3; i + 1 < COUNT; i += 2) b = max3(b, z[i], z[i + 1]);
  b = fmaxf(b, z[COUNT - 1]);
  a.largest = fmaxf(a.largest, b);
  if (b > a.m) rebase<ENT>(a, b, c2);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const float d = (z[i] - a.m) * c2, e = exp2_hw(d);
    a.s += e;
    if (ENT) a.t = __builtin_fmaf(e, fmaxf(d, -200.f), a.t);      // e is 0 there: keeps 0 * -infinity out
  }
}

template <int DT, int THREADS, bool ENT> __device__ inline RowSums sum_row(const Segment<DT>& row, float c2) {
  constexpr int N = Elem<DT>::N, U = 4;
  const int full = row.full(), items = row.items();
  RowSums a;
  int i = threadIdx.x;
  if (row.skew && i == 0) {
    float z[N];
    row.load(0, z);
    add_elements<N, ENT>(a, z, c2);
    i += THREADS;
  }
  for (; i + (U - 1) * THREADS < full; i += U * THREADS) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = row.vector(i + u * THREADS);
    float z[U * N];
#pragma unroll
    for (int u = 0; u < U; ++u) Elem<DT>::unpack(v[u], z + u * N);
    add_elements<U * N, ENT>(a, z, c2);
  }
  for (; i < items; i += THREADS) {
    float z[N];
    row.load(i, z);
    add_elements<N, ENT>(a, z, c2);
  }
  return a;
}

// The threads' sums of a row as one, in every thread.
template <int THREADS, bool ENT> __device__ inline RowSums join_row(RowSums a, float c2, float* lds) {
  RowSums r;
  r.largest = block_max<THREADS>(a.largest, lds);
  r.m = fmaxf(r.largest, kLowest);
  rebase<ENT>(a, r.m, c2);
  r.s = block_sum<THREADS>(a.s, lds);
  if (ENT) r.t = block_sum<THREADS>(a.t, lds);
  return r;
}

// ---- the k largest elements of a row ------------------------------------------------------------------
// Order: larger value first, lower place first among equals; NaN is never among them.  An element is
// a 64-bit key, its value's order (0: not a number) above its place counted from the end.

__device__ inline uint32_t order_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);              // -0 counts as +0
  if (z != z) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// (of order 0, the missing alternative of a row with NaN: NaN, and its place is -1)
__device__ inline float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ inline uint64_t key_of(uint32_t order, uint32_t place) { return static_cast<uint64_t>(order) << 32 | (0xffffffffu - place); }
__device__ inline uint32_t place_of(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }

template <int THREADS> struct Selection {
  uint32_t group[64];
  int count, owners;
  uint16_t owner[THREADS];
  uint64_t found[kCandidates];
  uint64_t top[kMaxTop];
};

// What is selected from is spread over the threads: item i of the source is thread i % THREADS's.  A
// source gives the (order, place) pairs of `U` items at a time, so that their loads overlap.

// A segment of a row by its items; `base` is the segment's place in its row.
template <int DT> struct RowSource {
  static constexpr int N = Elem<DT>::N, U = 2;
  Segment<DT> row;
  int base;
  __device__ int items() const { return row.items(); }
  template <class F> __device__ void visit(const int* item, F&& f) const {
    float z[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (item[u] >= 0) row.load(item[u], z[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (item[u] < 0) continue;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int at = row.place(item[u], j);
        if (const uint32_t order = order_of(z[u][j]); order && at >= 0 && at < row.n) f(order, static_cast<uint32_t>(base + at));
      }
    }
  }
};
// Keys in memory (0: none).
struct KeySource {
  static constexpr int U = 4;
  const uint64_t* keys;
  int n;
  __device__ int items() const { return n; }
  template <class F> __device__ void visit(const int* item, F&& f) const {
    uint64_t k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = item[u] >= 0 ? keys[item[u]] : 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k[u]) f(static_cast<uint32_t>(k[u] >> 32), place_of(k[u]));
  }
};
template <int THREADS, class Source, class F> __device__ inline void visit_own(const Source& src, F&& f) {
  const int items = src.items();
  for (int i = threadIdx.x; i < items; i += Source::U * THREADS) {
    int item[Source::U];
#pragma unroll
    for (int u = 0; u < Source::U; ++u) item[u] = i + u * THREADS < items ? i + u * THREADS : -1;
    src.visit(item, f);
  }
}

// Leaves the k largest keys of `src` in sel.top, largest first (0 behind the last where there are
// fewer).  `mine`: the largest order among the thread's own elements, 0 if it has none.
//
// The threads form 64 groups.  The k-th largest of the groups' maxima is no larger than the row's
// k-th largest element, so the k are among the elements at or above it, about as many as k in a
// row without structure: only the items of threads that have one are read again, by all threads
// together (by the thread itself that was 25 us of latency for a row of 50000, 3.4 us a row with
// eight rows on a compute unit).  A wave finds the threshold bit by bit with ballots.  A row with
// many elements there (equal ones, say) takes k rounds over the row instead.
template <int THREADS, class Source>
__device__ inline void select_top(const Source& src, uint32_t mine, int k, Selection<THREADS>& sel) {
  constexpr int G = THREADS / 64;
  uint32_t g = mine;
  if (G >= 2) g = max(g, dpp<kSwap1>(g, g));
  if (G >= 4) g = max(g, dpp<kSwap2>(g, g));
  if (G >= 8) g = max(g, dpp<kHalfMirror>(g, g));
  if (G >= 16) g = max(g, dpp<kMirror>(g, g));
  if (threadIdx.x % G == 0) sel.group[threadIdx.x / G] = g;
  if (threadIdx.x == 0) sel.count = sel.owners = 0;
  if (threadIdx.x < kMaxTop) sel.top[threadIdx.x] = 0;
  __syncthreads();
  g = sel.group[threadIdx.x & 63];
  uint32_t tau = 0;
#pragma unroll 1
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = tau | 1u << b;
    const int above = static_cast<int>(__popcll(__ballot(g >= t)));
    if (above >= k) tau = t;
    if (above == k) break;                                  // lower bits would not part the groups any more
  }
  if (mine && mine >= tau) sel.owner[atomicAdd(&sel.owners, 1)] = static_cast<uint16_t>(threadIdx.x);
  __syncthreads();
  const int owners = sel.owners, items = src.items(), total = owners * ((items + THREADS - 1) / THREADS);
  for (int i = threadIdx.x; i < total; i += Source::U * THREADS) {
    int item[Source::U];
#pragma unroll
    for (int u = 0; u < Source::U; ++u) {
      const int at = i + u * THREADS;
      item[u] = at < total ? sel.owner[at % owners] + at / owners * THREADS : -1;
      if (item[u] >= items) item[u] = -1;
    }
    src.visit(item, [&](uint32_t order, uint32_t place) {
      if (order >= tau) {
        const int found = atomicAdd(&sel.count, 1);
        if (found < kCandidates) sel.found[found] = key_of(order, place);
      }
    });
  }
  __syncthreads();
  const int count = sel.count;
  if (count <= kCandidates) {
    for (int i = threadIdx.x; i < count; i += THREADS) {
      const uint64_t key = sel.found[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j) rank += sel.found[j] > key;
      if (rank < k) sel.top[rank] = key;
    }
  } else {
    unsigned long long last = ~0ull;
    for (int r = 0; r < k; ++r) {
      unsigned long long b = 0;
      visit_own<THREADS>(src, [&](uint32_t order, uint32_t place) {
        const uint64_t key = key_of(order, place);
        if (key < last && key > b) b = key;
      });
      for (int off = 32; off > 0; off /= 2) b = max(b, __shfl_xor(b, off));
      __syncthreads();                                      // everybody has read the round before's
      if ((threadIdx.x & 63) == 0) sel.found[threadIdx.x / 64] = b;
      __syncthreads();
      last = sel.found[0];
      for (int w = 1; w < THREADS / 64; ++w) last = max(last, static_cast<unsigned long long>(sel.found[w]));
      if (threadIdx.x == 0) sel.top[r] = last;
    }
  }
  __syncthreads();
}
static_assert(kCandidates >= 1024 / 64, "the rounds over a row use a key per wave");

// ---- token log probabilities ---------------------------------------------------------------------------

// (a segment's sums go to the workspace as a Partial; its best keys follow all rows' partials)
typedef RowPartial Partial;

// The given token's logit; read ahead of the sums, so that nobody waits for it behind them.
struct Target {
  int64_t id;
  float z;
  __device__ Target(const ScoreArgs& a, int64_t row) : id(load_id(a.targets, row)), z(0.f) {
    if (id >= 0 && id < a.in.vocab) z = load_as(a.in.z, row * a.in.stride + id, a.in.dtype);
  }
};

// What a row reports, once its sums (and best keys) are known.  All threads of the workgroup call it.
__device__ inline void report_row(const ScoreArgs& a, int64_t row, const RowSums& r, const Target& target, const uint64_t* top) {
  const float scale = a.in.scale;
  const bool empty = r.s == 0.f;                            // no element above -infinity
  const float log_s = log2_hw(r.s) * kLn2;
  if (threadIdx.x == 0) {
    const int64_t id = target.id;
    float lp = 0.f;
    if (id != a.ignore) {
      lp = __builtin_nanf("");
      if (id >= 0 && id < a.in.vocab) lp = empty ? -INFINITY : (target.z - r.m) * scale - log_s;
    }
    a.logp[row] = lp;
    a.norm[2 * row] = r.largest;
    a.norm[2 * row + 1] = log_s;
    if (a.entropy) a.entropy[row] = empty ? 0.f : (log2_hw(r.s) - r.t / r.s) * kLn2;
  }
  const int j = threadIdx.x;
  if (a.top && j < a.top) {
    const uint64_t key = top[j];
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    a.top_ids[row * a.top + j] = static_cast<int>(place_of(key));
    a.top_logp[row * a.top + j] = empty ? -INFINITY : (value_of(order) - r.m) * scale - log_s;
  }
}

// A workgroup for each segment of each row; whole rows are reported at once.
template <int DT, int THREADS, bool ENT, bool TOP> __global__ __launch_bounds__(THREADS, THREADS == 1024 ? 4 : THREADS == 64 ? 6 : 8) void score_rows(ScoreArgs a) {
  __shared__ float lds[THREADS / 64];
  __shared__ typename std::conditional<TOP, Selection<THREADS>, char>::type sel;
  const int64_t row = blockIdx.x / a.split.segs;
  const int seg = blockIdx.x % a.split.segs, lo = seg * a.split.seg;
  const int n = min(a.split.seg, a.in.vocab - lo);
  const auto* p = static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride + lo;
  const float c2 = a.in.scale * kLog2e;
  const Target target(a, row);
  const Segment<DT> part(p, n);
  const RowSums mine = sum_row<DT, THREADS, ENT>(part, c2);
  const RowSums r = join_row<THREADS, ENT>(mine, c2, lds);
  if constexpr (TOP) {
    const bool has = static_cast<int>(threadIdx.x) < part.items();
    select_top<THREADS>(RowSource<DT>{part, lo}, has ? order_of(mine.largest) : 0u, a.top, sel);
  }
  if (a.split.segs == 1) {
    if constexpr (TOP) report_row(a, row, r, target, sel.top);
    else report_row(a, row, r, target, nullptr);
    return;
  }
  Partial* parts = static_cast<Partial*>(a.workspace);
  if (threadIdx.x == 0) parts[blockIdx.x] = {r.largest, r.s, r.t, 0.f};
  if constexpr (TOP) {
    uint64_t* keys = reinterpret_cast<uint64_t*>(parts + a.in.rows * a.split.segs);
    if (static_cast<int>(threadIdx.x) < a.top) keys[static_cast<int64_t>(blockIdx.x) * a.top + threadIdx.x] = sel.top[threadIdx.x];
  }
}

// Rows without alternatives of up to kScoreHeld items a thread, held in registers from one reading: all loads are
// under way at once, the sums are relative to the row's own maximum and no thread's has to be moved.  16384 x
// 8000 bf16 39 us (6.7 TB/s, read again from partly warm caches) where the kernel above takes 50.  Without the bound of four
// waves a SIMD the compiler takes 82 registers for f32, and 8192 x 8000 f32 43 us instead of 37.  (With
// alternatives it would be slower, 91 us instead of 59: the selection from registers takes twice as many of them.)
template <int DT, int THREADS, int NV, bool ENT> __global__ __launch_bounds__(THREADS, 4) void score_held(ScoreArgs a) {
  constexpr int N = Elem<DT>::N, W = THREADS / 64;
  __shared__ float most[W], sums[2 * W];
  const int64_t row = blockIdx.x;
  const Segment<DT> part(static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride, a.in.vocab);
  const Target target(a, row);
  const int full = part.full(), wave = threadIdx.x >> 6;
  u32x4 v[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int i = threadIdx.x + u * THREADS;
    if (i < full && (i > 0 || part.skew == 0)) v[u] = part.vector(i);
  }
  float z[NV * N];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int i = threadIdx.x + u * THREADS;
    if (i < full && (i > 0 || part.skew == 0)) {
      Elem<DT>::unpack(v[u], z + u * N);
    } else {
      part.load(i, z + u * N);                              // an end of the row, or nothing of it
    }
  }
  float mine = z[0];
#pragma unroll
  for (int i = 1; i + 1 < NV * N; i += 2) mine = max3(mine, z[i], z[i + 1]);
  const float wave_most = wave_max(fmaxf(mine, z[NV * N - 1]));
  if ((threadIdx.x & 63) == 0) most[wave] = wave_most;
  __syncthreads();
  RowSums r;
  r.largest = most[0];
#pragma unroll
  for (int w = 1; w < W; ++w) r.largest = fmaxf(r.largest, most[w]);
  r.m = fmaxf(r.largest, kLowest);
  const float c2 = a.in.scale * kLog2e;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < NV * N; ++i) {
    const float d = (z[i] - r.m) * c2, e = exp2_hw(d);
    s += e;
    if (ENT) t = __builtin_fmaf(e, fmaxf(d, -200.f), t);
  }
  s = wave_sum(s);
  if (ENT) t = wave_sum(t);
  if ((threadIdx.x & 63) == 0) sums[wave] = s, sums[W + wave] = t;
  __syncthreads();
  r.s = sums[0], r.t = sums[W];
#pragma unroll
  for (int w = 1; w < W; ++w) r.s += sums[w], r.t += sums[W + w];
  report_row(a, row, r, target, nullptr);
}

// This thread's share of the sums of a row's segments.
template <int THREADS, bool ENT> __device__ inline RowSums add_parts(const Partial* parts, int segs, float c2) {
  RowSums a;
  for (int i = threadIdx.x; i < segs; i += THREADS) {
    const Partial p = parts[i];
    RowSums b;
    b.largest = p.largest, b.m = fmaxf(p.largest, kLowest), b.s = p.s, b.t = p.t;
    const float m = fmaxf(a.m, b.m);
    rebase<ENT>(a, m, c2);
    rebase<ENT>(b, m, c2);
    a.largest = fmaxf(a.largest, b.largest);
    a.s += b.s;
    a.t += b.t;
  }
  return a;
}

template <int THREADS, bool ENT, bool TOP> __global__ __launch_bounds__(THREADS) void score_join(ScoreArgs a) {
  __shared__ float lds[THREADS / 64];
  __shared__ typename std::conditional<TOP, Selection<THREADS>, char>::type sel;
  const int64_t row = blockIdx.x;
  const int segs = a.split.segs;
  const Partial* parts = static_cast<const Partial*>(a.workspace);
  const Target target(a, row);
  const RowSums r = join_row<THREADS, ENT>(add_parts<THREADS, ENT>(parts + row * segs, segs, a.in.scale * kLog2e), a.in.scale * kLog2e, lds);
  if constexpr (TOP) {
    const uint64_t* keys = reinterpret_cast<const uint64_t*>(parts + a.in.rows * segs) + row * segs * a.top;
    const KeySource src{keys, segs * a.top};
    uint32_t mine = 0;
    visit_own<THREADS>(src, [&](uint32_t order, uint32_t) { mine = max(mine, order); });
    select_top<THREADS>(src, mine, a.top, sel);
    report_row(a, row, r, target, sel.top);
  } else {
    report_row(a, row, r, target, nullptr);
  }
}

// dz_i = c [ g ([i = t] - p_i) - e p_i (log p_i + H) ] with g, e the gradients of log p_t and H: one
// pass, a vector for each thread.  Workgroups of 4 KB keep what is on the way in memory order:
// 8192 x 65536 bf16 in 389 us (5.5 TB/s; a copy of as much reaches 5.0); more vectors a thread, or a row for a
// workgroup, were 7 and 20% slower.
template <int DT, bool ENT> __global__ __launch_bounds__(256) void score_grad_rows(ScoreGradArgs a, int spans, int64_t row0) {
  constexpr int N = Elem<DT>::N;
  typedef typename Elem<DT>::T T;
  const int64_t row = row0 + blockIdx.x / spans;
  const int at = (static_cast<int>(blockIdx.x % spans) * 256 + static_cast<int>(threadIdx.x)) * N, n = a.in.vocab - at;
  if (n <= 0) return;
  const T* p = static_cast<const T*>(a.in.z) + row * a.in.stride + at;
  T* out = static_cast<T*>(a.grad) + row * a.grad_stride + at;
  float z[N];
  if (n >= N) {
    Elem<DT>::unpack(load16(p), z);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = j < n ? Elem<DT>::get(p[j]) : 0.f;
  }
  const float m = a.norm[2 * row], log_s = a.norm[2 * row + 1], scale = a.in.scale;
  const bool empty = m == -INFINITY && log_s == -INFINITY;
  const int64_t id = load_id(a.targets, row);
  float g = a.grad_logp ? a.grad_logp[row] : 0.f;
  const float e = ENT ? a.grad_entropy[row] : 0.f;
  if (id == a.ignore) g = 0.f;
  else if (id < 0 || id >= a.in.vocab) g = __builtin_nanf("");
  const float all = scale * (ENT ? g + e * a.entropy[row] : g), each = scale * e;
  const int64_t target = id == a.ignore || empty ? -1 : id - at;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float lp = (z[j] - m) * scale - log_s, pr = exp2_hw(lp * kLog2e);
    z[j] = empty ? 0.f : ENT ? -pr * (all + each * fmaxf(lp, -200.f)) : -pr * all;
    if (j == target) z[j] += scale * g;
  }
  if (n >= N) {
    stream16(out, Elem<DT>::pack(z));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) out[j] = Elem<DT>::put(z[j]);
  }
}

// ---- distillation --------------------------------------------------------------------------------------

// The teacher's entries of a row, in as much LDS as they need, and for each thread the chain of those
// whose elements it writes.
struct Teacher {
  int* ids;                      // -1: no entry
  int* next;                     // the next entry of the same owner, -1 behind the last
  float* q;
  float* log_q;
  float* sum;                    // q of all entries that name the same token: one named twice counts twice
  float* z;                      // the student's logit
  int* head;                     // a thread's first entry, -1: none
  __device__ Teacher(float* lds, int k)
      : ids(reinterpret_cast<int*>(lds)), next(ids + k), q(lds + 2 * k), log_q(lds + 3 * k), sum(lds + 4 * k), z(lds + 5 * k),
        head(ids + 6 * k) {}
  __host__ __device__ static size_t bytes16(int k, int threads) { return (24 * static_cast<size_t>(k) + 4 * static_cast<size_t>(threads) + 15) / 16 * 16; }
  static size_t bytes(int k, int threads) { return 24 * static_cast<size_t>(k) + 4 * static_cast<size_t>(threads); }
};
extern __shared__ float teacher_lds[];

// A thread's first entry while it is on its way from memory.
struct Entry {
  int id;
  float u;
  __device__ Entry(const DistillArgs& a, int64_t row, int k) : id(-1), u(-INFINITY) {
    if (k >= a.k) return;
    const int64_t i = load_id(a.ids, row * a.ids_stride + k);
    u = load_as(a.teacher, row * a.teacher_stride + k, a.teacher_dtype);
    if (i >= 0 && i < a.in.vocab) id = static_cast<int>(i);
  }
};

// The teacher's probabilities of a row into LDS: sum q is 1, or 0 where no entry has any, and is
// returned.  Entries whose id is not a token have none.  OWNERS: the chains too; element i is written
// by the thread that has vector i / N, behind the last whole vector by thread i - N * full.
template <int THREADS, int N, bool OWNERS>
__device__ inline float load_teacher(const DistillArgs& a, int64_t row, const Entry& first, const Teacher& t, float* lds) {
  const float inv = 1.f / a.temperature;
  if (OWNERS) t.head[threadIdx.x] = -1;
  float m = -INFINITY;
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const Entry e = k < THREADS ? first : Entry(a, row, k);
    const float u = e.id >= 0 ? e.u : -INFINITY;
    t.ids[k] = e.id;
    t.q[k] = u;
    m = u != u ? u : fmaxf(m, u);
  }
  m = fmaxf(block_max<THREADS>(m, lds), kLowest);
  float s = 0.f;
  for (int k = threadIdx.x; k < a.k; k += THREADS)
    if (t.ids[k] >= 0) s += exp2_hw((t.q[k] - m) * inv * kLog2e);
  s = block_sum<THREADS>(s, lds);
  const float log_s = log2_hw(s) * kLn2;
  const bool none = s == 0.f;
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const float log_q = (t.q[k] - m) * inv - log_s;
    t.log_q[k] = log_q;
    t.q[k] = t.ids[k] >= 0 && !none ? exp2_hw(log_q * kLog2e) : 0.f;
    if (OWNERS && t.ids[k] >= 0) {
      const int id = t.ids[k], full = a.in.vocab / N;
      t.next[k] = atomicExch(&t.head[id < full * N ? id / N % THREADS : id - full * N], k);
    }
  }
  __syncthreads();
  if (OWNERS)
    for (int k = threadIdx.x; k < a.k; k += THREADS) {
      float sum = 0.f;
      for (int j = 0; j < a.k; ++j) sum += t.ids[j] == t.ids[k] ? t.q[j] : 0.f;
      t.sum[k] = sum;
    }
  return none ? 0.f : 1.f;
}

template <int DT> __device__ inline float student(const DistillArgs& a, int64_t row, int id) {
  return id >= 0 ? Elem<DT>::get(static_cast<const typename Elem<DT>::T*>(a.in.z)[row * a.in.stride + id]) : 0.f;
}

// The threads' sums of a row as one, and the row's loss and statistics reported:
// T^2 sum_k q_k (log q_k - log p_(id_k)), the sum without log S taken along with S itself.
// `zk`: the student's logit of the thread's first entry.
template <int DT, int THREADS>
__device__ inline RowSums join_and_report(const DistillArgs& a, int64_t row, RowSums mine, float zk, float total, const Teacher& t, float* lds) {
  const float c2 = a.in.scale * kLog2e;
  RowSums r;
  r.largest = block_max<THREADS>(mine.largest, lds);
  r.m = fmaxf(r.largest, kLowest);
  rebase<false>(mine, r.m, c2);
  r.s = mine.s;
  float kl = 0.f;
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const float q = t.q[k], z = k < THREADS ? zk : student<DT>(a, row, t.ids[k]);
    t.z[k] = z;
    if (q != 0.f) kl += q * (t.log_q[k] - (z - r.m) * a.in.scale);
  }
  block_sum<THREADS>(r.s, kl, lds);
  if (threadIdx.x == 0) {
    const float log_s = log2_hw(r.s) * kLn2;
    if (r.s == 0.f) kl = INFINITY;
    else kl += log_s;
    // (a row without entries may hold anything, NaN among it)
    a.loss[row] = total != 0.f ? kl * a.temperature * a.temperature : 0.f;
    a.norm[2 * row] = r.largest;
    a.norm[2 * row + 1] = log_s;
  }
  return r;
}

// dz_i = w T (p_i - sum_{k: id_k = i} q_k) with p_i = exp2(c2 (z_i - m) - log2 S), in rows that have entries.
struct Gradient {
  float w, m, c2, shift;
  __device__ Gradient(const DistillArgs& a, int64_t row, float m_, float log2_s, bool empty)
      : w(empty ? 0.f : (a.weight ? a.weight[row] : 1.f) * a.temperature), m(empty ? INFINITY : m_), c2(a.in.scale * kLog2e),
        shift(empty ? 0.f : log2_s) {}
  // from the pair that the loss left
  __device__ Gradient(const DistillArgs& a, int64_t row)
      : Gradient(a, row, a.norm[2 * row], a.norm[2 * row + 1] * kLog2e, a.norm[2 * row] == -INFINITY && a.norm[2 * row + 1] == -INFINITY) {}
  __device__ float operator()(float z) const { return w * exp2_hw(__builtin_fmaf(z - m, c2, -shift)); }
};

// The entries that the teacher names, by the threads that have written those elements without them: a
// thread's stores to one address stay in order.
template <int DT>
__device__ inline void write_named(const Teacher& t, const Gradient& g, typename Elem<DT>::T* out) {
  for (int k = t.head[threadIdx.x]; k >= 0; k = t.next[k]) out[t.ids[k]] = Elem<DT>::put(g(t.z[k]) - g.w * t.sum[k]);
}

// The gradient of a row without entries, whatever its logits are.
template <int DT, int THREADS> __device__ inline void clear_row(typename Elem<DT>::T* out, int n) {
  constexpr int N = Elem<DT>::N;
  const int full = n / N;
  for (int i = threadIdx.x; i < full; i += THREADS) store16(out + static_cast<int64_t>(i) * N, u32x4{0, 0, 0, 0});
  if (const int i = full * N + static_cast<int>(threadIdx.x); i < n) out[i] = Elem<DT>::put(0.f);
}

// A row to a workgroup, in its registers (THREADS * NV vectors) from one reading: the loss and the
// gradient.  What concerns the teacher is found while the logits arrive.  Bound by memory, with one
// row of 250 KB on a compute unit by the waits between its reading and its writing too: 8192 x 128000
// bf16 in 829 us (5.1 TB/s).  Read a second time instead: 1280 us with four times as many rows on the
// way as the last-level cache holds, 950 us with as many as it does hold.
// EX: vectors a thread keeps in LDS besides, read first, while the registers are free (3000 x 80000 f32 376 us;
// with two readings, the loss and then the gradient from what it leaves, 480).
template <int DT, int THREADS, int NV, int EX> __global__ __launch_bounds__(THREADS, 4) void distill_held(DistillArgs a) {
  constexpr int N = Elem<DT>::N;
  typedef typename Elem<DT>::T T;
  __shared__ float lds[2 * THREADS / 64];
  const Teacher teacher(teacher_lds, a.k);
  const int64_t row = blockIdx.x;
  const int n = a.in.vocab, full = n / N, rest = n % N;
  const T* p = static_cast<const T*>(a.in.z) + row * a.in.stride;
  T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
  const Entry first(a, row, threadIdx.x);
  const u32x4 nothing = {Elem<DT>::kMinusInfinity, Elem<DT>::kMinusInfinity, Elem<DT>::kMinusInfinity, Elem<DT>::kMinusInfinity};
  u32x4* kept = reinterpret_cast<u32x4*>(reinterpret_cast<char*>(teacher_lds) + Teacher::bytes16(a.k, THREADS)) + threadIdx.x;
  if constexpr (EX > 0) {
    u32x4 v[EX];
#pragma unroll
    for (int i = 0; i < EX; ++i) {
      const int at = (NV + i) * THREADS + static_cast<int>(threadIdx.x);
      v[i] = nothing;
      if (at < full) v[i] = load16(p + at * N);
    }
#pragma unroll
    for (int i = 0; i < EX; ++i) kept[i * THREADS] = v[i];
    __builtin_amdgcn_sched_barrier(0);                      // the other loads need these registers
  }
  u32x4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = i * THREADS + static_cast<int>(threadIdx.x);
    v[i] = nothing;
    if (at < full) v[i] = load16(p + at * N);
  }
  const bool tail = static_cast<int>(threadIdx.x) < rest;
  const float last = tail ? Elem<DT>::get(p[full * N + threadIdx.x]) : -INFINITY;
  const float zk = student<DT>(a, row, first.id);
  const float total = load_teacher<THREADS, N, true>(a, row, first, teacher, lds);
  const float c2 = a.in.scale * kLog2e;
  RowSums mine;
#pragma unroll
  for (int i = 0; i < NV; i += 2) {
    if (i * THREADS >= full) break;
    float z[2 * N];
    Elem<DT>::unpack(v[i], z);
    Elem<DT>::unpack(v[i + 1], z + N);
    add_elements<2 * N, false>(mine, z, c2);
  }
#pragma unroll 1
  for (int i = 0; i < EX; i += 2) {
    float z[2 * N];
    Elem<DT>::unpack(kept[i * THREADS], z);
    Elem<DT>::unpack(kept[(i + 1) * THREADS], z + N);
    add_elements<2 * N, false>(mine, z, c2);
  }
  const float z[4] = {last, -INFINITY, -INFINITY, -INFINITY};
  add_elements<4, false>(mine, z, c2);
  const RowSums r = join_and_report<DT, THREADS>(a, row, mine, zk, total, teacher, lds);
  if (total == 0.f) {
    clear_row<DT, THREADS>(out, n);
    return;
  }
  const Gradient gradient(a, row, r.m, log2_hw(r.s), r.s == 0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * THREADS >= full) break;
    const int at = i * THREADS + static_cast<int>(threadIdx.x);
    float z[N];
    Elem<DT>::unpack(v[i], z);
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = gradient(z[j]);
    if (at < full) store16(out + at * N, Elem<DT>::pack(z));
  }
#pragma unroll 1
  for (int i = 0; i < EX; ++i) {
    const int at = (NV + i) * THREADS + static_cast<int>(threadIdx.x);
    if (at >= full) break;
    float z[N];
    Elem<DT>::unpack(kept[i * THREADS], z);
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = gradient(z[j]);
    store16(out + at * N, Elem<DT>::pack(z));
  }
  if (tail) out[full * N + threadIdx.x] = Elem<DT>::put(gradient(last));
  write_named<DT>(teacher, gradient, out);
}

// The gradient from the pair (m, log S) that the loss left, in two launches: all elements as if the
// teacher named none of them, a vector a thread in memory order, then a workgroup a row for those
// that it does name (and for rows where it names none at all, whose gradient is 0).
template <int DT> __global__ __launch_bounds__(256) void distill_stream(DistillArgs a, int spans, int64_t row0) {
  constexpr int N = Elem<DT>::N;
  typedef typename Elem<DT>::T T;
  const int64_t row = row0 + blockIdx.x / spans;
  const int at = (static_cast<int>(blockIdx.x % spans) * 256 + static_cast<int>(threadIdx.x)) * N, n = a.in.vocab - at;
  if (n <= 0) return;
  const T* p = static_cast<const T*>(a.in.z) + row * a.in.stride + at;
  T* out = static_cast<T*>(a.grad) + row * a.grad_stride + at;
  float z[N];
  if (n >= N) {
    Elem<DT>::unpack(load16(p), z);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = j < n ? Elem<DT>::get(p[j]) : 0.f;
  }
  const Gradient gradient(a, row);
#pragma unroll
  for (int j = 0; j < N; ++j) z[j] = gradient(z[j]);
  if (n >= N) {
    stream16(out, Elem<DT>::pack(z));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) out[j] = Elem<DT>::put(z[j]);
  }
}
template <int DT, int THREADS> __global__ __launch_bounds__(THREADS) void distill_named(DistillArgs a) {
  __shared__ float lds[THREADS / 64];
  const Teacher teacher(teacher_lds, a.k);
  const int64_t row = blockIdx.x;
  const Entry first(a, row, threadIdx.x);
  const float zk = student<DT>(a, row, first.id);
  const float total = load_teacher<THREADS, Elem<DT>::N, true>(a, row, first, teacher, lds);
  auto* out = static_cast<typename Elem<DT>::T*>(a.grad) + row * a.grad_stride;
  if (total == 0.f) {
    clear_row<DT, THREADS>(out, a.in.vocab);
    return;
  }
  const Gradient gradient(a, row);
  for (int k = threadIdx.x; k < a.k; k += THREADS)
    if (const int id = teacher.ids[k]; id >= 0)
      out[id] = Elem<DT>::put(gradient(k < THREADS ? zk : student<DT>(a, row, id)) - gradient.w * teacher.sum[k]);
}

// The loss alone.
template <int DT, int THREADS> __global__ __launch_bounds__(THREADS) void distill_rows(DistillArgs a) {
  __shared__ float lds[2 * THREADS / 64];
  const Teacher teacher(teacher_lds, a.k);
  const int64_t row = blockIdx.x;
  const Segment<DT> part(static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride, a.in.vocab);
  const Entry first(a, row, threadIdx.x);
  const float zk = student<DT>(a, row, first.id);
  const float total = load_teacher<THREADS, Elem<DT>::N, false>(a, row, first, teacher, lds);
  join_and_report<DT, THREADS>(a, row, sum_row<DT, THREADS, false>(part, a.in.scale * kLog2e), zk, total, teacher, lds);
}

// Few rows that are long: segments' sums, then a workgroup a row joins them and finds the loss.
template <int DT, int THREADS> __global__ __launch_bounds__(THREADS) void distill_parts(DistillArgs a) {
  __shared__ float lds[THREADS / 64];
  const int64_t row = blockIdx.x / a.split.segs;
  const int lo = static_cast<int>(blockIdx.x % a.split.segs) * a.split.seg, n = min(a.split.seg, a.in.vocab - lo);
  const auto* p = static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride + lo;
  const float c2 = a.in.scale * kLog2e;
  const RowSums r = join_row<THREADS, false>(sum_row<DT, THREADS, false>(Segment<DT>(p, n), c2), c2, lds);
  if (threadIdx.x == 0) static_cast<Partial*>(a.workspace)[blockIdx.x] = {r.largest, r.s, 0.f, 0.f};
}
template <int DT, int THREADS> __global__ __launch_bounds__(THREADS) void distill_join(DistillArgs a) {
  __shared__ float lds[2 * THREADS / 64];
  const Teacher teacher(teacher_lds, a.k);
  const int64_t row = blockIdx.x;
  const Entry first(a, row, threadIdx.x);
  const float zk = student<DT>(a, row, first.id);
  const float total = load_teacher<THREADS, Elem<DT>::N, false>(a, row, first, teacher, lds);
  const RowSums mine = add_parts<THREADS, false>(static_cast<const Partial*>(a.workspace) + row * a.split.segs, a.split.segs, a.in.scale * kLog2e);
  join_and_report<DT, THREADS>(a, row, mine, zk, total, teacher, lds);
}

template <class F> hipError_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f(std::integral_constant<int, kF32>{});
    case kBF16: return f(std::integral_constant<int, kBF16>{});
    default: return f(std::integral_constant<int, kF16>{});
  }
}
template <class F> hipError_t by_threads(int threads, F&& f) {
  switch (threads) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    case 512: return f(std::integral_constant<int, 512>{});
    default: return f(std::integral_constant<int, 1024>{});
  }
}
template <class F> hipError_t by_items(int items, F&& f) {
  switch (items) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    default: return f(std::integral_constant<int, kScoreHeld>{});
  }
}
template <int N> using Int = std::integral_constant<int, N>;
unsigned grid_of(int64_t n) { return static_cast<unsigned>(n); }
// `spans` workgroups for each row, in launches of as many rows as one can have.
template <class F> hipError_t by_row_runs(int64_t rows, int spans, F&& f) {
  const int64_t run = kLaunchBlocks / spans;
  for (int64_t row0 = 0; row0 < rows; row0 += run) {
    if (hipError_t e = f(row0, grid_of((rows - row0 < run ? rows - row0 : run) * spans))) return e;
  }
  return hipSuccess;
}

template <int DT> hipError_t launch_gradient_alone(const DistillArgs& a, hipStream_t stream) {
  constexpr int span = 256 * Elem<DT>::N;
  const int spans = (a.in.vocab + span - 1) / span;
  const hipError_t e = by_row_runs(a.in.rows, spans, [&](int64_t row0, unsigned grid) { return queue(distill_stream<DT>, grid, 256, 0, stream, a, spans, row0); });
  if (e != hipSuccess) return e;
  if (a.k <= 64) return queue(distill_named<DT, 64>, grid_of(a.in.rows), 64, Teacher::bytes(a.k, 64), stream, a);
  return queue(distill_named<DT, 256>, grid_of(a.in.rows), 256, Teacher::bytes(a.k, 256), stream, a);
}

}  // namespace

hipError_t launch_score(const ScoreArgs& a, hipStream_t stream) {
  auto go = [&](auto dt, auto ent, auto top) {
    hipError_t e = by_threads(a.split.threads, [&](auto threads) {
      if constexpr (!top.value) {
        if (a.split.held) {
          return by_items(a.split.held, [&](auto items) {
            if constexpr (held_form(threads.value, items.value))
              return queue(score_held<dt.value, threads.value, items.value, ent.value>, grid_of(a.in.rows), threads.value, 0, stream, a);
            else return hipErrorInvalidValue;
          });
        }
      }
      // (shorter rows without alternatives are held)
      if constexpr (top.value || threads.value >= 256)
        return queue(score_rows<dt.value, threads.value, ent.value, top.value>, grid_of(a.in.rows * a.split.segs), threads.value, 0, stream, a);
      else return hipErrorInvalidValue;
    });
    if (e != hipSuccess || a.split.segs == 1) return e;
    return queue(score_join<256, ent.value, top.value>, grid_of(a.in.rows), 256, 0, stream, a);
  };
  return by_type(a.in.dtype, [&](auto dt) {
    const std::true_type yes;
    const std::false_type no;
    if (a.entropy) return a.top ? go(dt, yes, yes) : go(dt, yes, no);
    return a.top ? go(dt, no, yes) : go(dt, no, no);
  });
}

hipError_t launch_score_grad(const ScoreGradArgs& a, hipStream_t stream) {
  return by_type(a.in.dtype, [&](auto dt) {
    constexpr int span = 256 * Elem<dt.value>::N;
    const int spans = (a.in.vocab + span - 1) / span;
    return by_row_runs(a.in.rows, spans, [&](int64_t row0, unsigned grid) {
      if (a.grad_entropy) return queue(score_grad_rows<dt.value, true>, grid, 256, 0, stream, a, spans, row0);
      return queue(score_grad_rows<dt.value, false>, grid, 256, 0, stream, a, spans, row0);
    });
  });
}

hipError_t launch_distill_grad(const DistillArgs& a, hipStream_t stream) {
  return by_type(a.in.dtype, [&](auto dt) { return launch_gradient_alone<dt.value>(a, stream); });
}

hipError_t launch_distill(const DistillArgs& a, hipStream_t stream) {
  return by_type(a.in.dtype, [&](auto dt) {
    constexpr int DT = dt.value;
    const unsigned rows = grid_of(a.in.rows);
    if (a.split.segs > 1) {
      if (hipError_t e = queue(distill_parts<DT, 512>, grid_of(a.in.rows * a.split.segs), 512, 0, stream, a)) return e;
      const hipError_t e = queue(distill_join<DT, 256>, rows, 256, Teacher::bytes(a.k, 256), stream, a);
      return e != hipSuccess || !a.grad ? e : launch_gradient_alone<DT>(a, stream);
    }
    if (!a.grad || a.held.vectors == 0) {
      const hipError_t e = by_threads(a.split.threads, [&](auto threads) {
        return queue(distill_rows<DT, threads.value>, rows, threads.value, Teacher::bytes(a.k, threads.value), stream, a);
      });
      return e != hipSuccess || !a.grad ? e : launch_gradient_alone<DT>(a, stream);
    }
    auto held = [&](auto threads, auto nv) {
      return queue(distill_held<DT, threads.value, nv.value, 0>, rows, threads.value, Teacher::bytes(a.k, threads.value), stream, a);
    };
    const RowHeld h = a.held;
    if (h.vectors == 4) {
      if (h.threads == 64) return held(Int<64>{}, Int<4>{});
      if (h.threads == 128) return held(Int<128>{}, Int<4>{});
      if (h.threads == 256) return held(Int<256>{}, Int<4>{});
      return held(Int<1024>{}, Int<4>{});
    }
    if (h.vectors == 8) return held(Int<256>{}, Int<8>{});
    if (h.vectors == 16) {
      if (h.threads == 256) return held(Int<256>{}, Int<16>{});
      if (h.threads == 512) return held(Int<512>{}, Int<16>{});
      return held(Int<1024>{}, Int<16>{});
    }
    return queue(distill_held<DT, 1024, 16, kHeldInLds>, rows, 1024, Teacher::bytes16(a.k, 1024) + 16 * 1024 * kHeldInLds, stream, a);
  });
}

}  // namespace eh
