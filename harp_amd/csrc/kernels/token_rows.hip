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
constexpr int kCandidates = 512;          // elements at or above the selection's threshold that LDS holds

__device__ inline int row_vectors(int n, int per) { return (n + per - 1) / per; }

// Elements [N * i, N * i + N) of a row's segment of n elements; those at n and behind are -infinity.
template <int DT> __device__ inline void load_vector(const typename Elem<DT>::T* p, int i, int n, float* z) {
  constexpr int N = Elem<DT>::N;
  if ((i + 1) * N <= n) {
    Elem<DT>::unpack(load16(p + static_cast<int64_t>(i) * N), z);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = i * N + j < n ? Elem<DT>::get(p[i * N + j]) : -INFINITY;
  }
}

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

template <int DT, int THREADS, bool ENT> __device__ inline RowSums sum_row(const typename Elem<DT>::T* p, int n, float c2) {
  constexpr int N = Elem<DT>::N, U = 4;
  const int full = n / N, all = row_vectors(n, N);
  RowSums a;
  int i = threadIdx.x;
  for (; i + (U - 1) * THREADS < full; i += U * THREADS) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(p + static_cast<int64_t>(i + u * THREADS) * N);
    float z[U * N];
#pragma unroll
    for (int u = 0; u < U; ++u) Elem<DT>::unpack(v[u], z + u * N);
    add_elements<U * N, ENT>(a, z, c2);
  }
  for (; i < all; i += THREADS) {
    float z[N];
    load_vector<DT>(p, i, n, z);
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

struct Selection {
  uint32_t group[64];
  int count;
  uint64_t found[kCandidates];
  uint64_t top[kMaxTop];
};

// A segment of a row: thread t has vectors t, t + THREADS, ...  `base` is the segment's place in its row.
template <int DT, int THREADS> struct RowSource {
  const typename Elem<DT>::T* p;
  int n, base;
  template <class F> __device__ void each(F&& f) const {
    constexpr int N = Elem<DT>::N;
    const int all = row_vectors(n, N);
    for (int i = threadIdx.x; i < all; i += THREADS) {
      float z[N];
      load_vector<DT>(p, i, n, z);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (const uint32_t order = order_of(z[j]); order && i * N + j < n) f(order, static_cast<uint32_t>(base + i * N + j));
    }
  }
};
// Keys in memory (0: none).
template <int THREADS> struct KeySource {
  const uint64_t* keys;
  int n;
  template <class F> __device__ void each(F&& f) const {
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const uint64_t k = keys[i];
      if (k) f(static_cast<uint32_t>(k >> 32), place_of(k));
    }
  }
};

// Leaves the k largest keys of `src` in sel.top, largest first (0 behind the last where there are
// fewer).  `mine`: the largest order among the thread's own elements, 0 if it has none.
//
// The threads form 64 groups.  The k-th largest of the groups' maxima is no larger than the row's
// k-th largest element, so the k are among the elements at or above it, about as many as k in a
// row without structure: only threads that have one read theirs again.  A wave finds that
// threshold bit by bit with ballots.  A row with many elements there (equal ones, say) takes k
// rounds over the row instead.
template <int THREADS, class Source>
__device__ inline void select_top(const Source& src, uint32_t mine, int k, Selection& sel) {
  constexpr int G = THREADS / 64;
  uint32_t g = mine;
  if (G >= 2) g = max(g, dpp<kSwap1>(g, g));
  if (G >= 4) g = max(g, dpp<kSwap2>(g, g));
  if (G >= 8) g = max(g, dpp<kHalfMirror>(g, g));
  if (G >= 16) g = max(g, dpp<kMirror>(g, g));
  if (threadIdx.x % G == 0) sel.group[threadIdx.x / G] = g;
  if (threadIdx.x == 0) sel.count = 0;
  if (threadIdx.x < kMaxTop) sel.top[threadIdx.x] = 0;
  __syncthreads();
  g = sel.group[threadIdx.x & 63];
  uint32_t tau = 0;
#pragma unroll 1
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = tau | 1u << b;
    if (static_cast<int>(__popcll(__ballot(g >= t))) >= k) tau = t;
  }
  if (mine && mine >= tau)
    src.each([&](uint32_t order, uint32_t place) {
      if (order >= tau) {
        const int at = atomicAdd(&sel.count, 1);
        if (at < kCandidates) sel.found[at] = key_of(order, place);
      }
    });
  __syncthreads();
  const int count = sel.count;
  if (count <= kCandidates) {
    for (int i = threadIdx.x; i < count; i += THREADS) {
      const uint64_t key = sel.found[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += sel.found[j] > key;
      if (rank < k) sel.top[rank] = key;
    }
  } else {
    uint64_t last = ~uint64_t{0};
    uint64_t* best = sel.found;
    for (int r = 0; r < k; ++r) {
      uint64_t b = 0;
      src.each([&](uint32_t order, uint32_t place) {
        const uint64_t key = key_of(order, place);
        if (key < last && key > b) b = key;
      });
      __syncthreads();
      best[threadIdx.x] = b;
      __syncthreads();
      for (int h = THREADS / 2; h > 0; h >>= 1) {
        if (static_cast<int>(threadIdx.x) < h && best[threadIdx.x + h] > best[threadIdx.x]) best[threadIdx.x] = best[threadIdx.x + h];
        __syncthreads();
      }
      last = best[0];
      if (threadIdx.x == 0) sel.top[r] = last;
    }
  }
  __syncthreads();
}
static_assert(kCandidates >= 512, "the rounds over a row use a key per thread");

// ---- token log probabilities ---------------------------------------------------------------------------

struct Partial {                 // a segment's sums; its best keys follow all rows' partials
  float largest, s, t, pad;
};

// What a row reports, once its sums (and best keys) are known.  All threads of the workgroup call it.
__device__ inline void report_row(const ScoreArgs& a, int64_t row, const RowSums& r, const Selection* sel) {
  const float scale = a.in.scale;
  const bool empty = r.s == 0.f;                            // no element above -infinity
  const float log_s = log2_hw(r.s) * kLn2;
  if (threadIdx.x == 0) {
    const int64_t id = load_id(a.targets, row);
    float lp = 0.f;
    if (id != a.ignore) {
      lp = __builtin_nanf("");
      if (id >= 0 && id < a.in.vocab)
        lp = empty ? -INFINITY : (load_as(a.in.z, row * a.in.stride + id, a.in.dtype) - r.m) * scale - log_s;
    }
    a.logp[row] = lp;
    a.norm[2 * row] = r.largest;
    a.norm[2 * row + 1] = log_s;
    if (a.entropy) a.entropy[row] = empty ? 0.f : (log2_hw(r.s) - r.t / r.s) * kLn2;
  }
  const int j = threadIdx.x;
  if (a.top && j < a.top) {
    const uint64_t key = sel->top[j];
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    a.top_ids[row * a.top + j] = static_cast<int>(place_of(key));
    a.top_logp[row * a.top + j] = empty ? -INFINITY : (value_of(order) - r.m) * scale - log_s;
  }
}

// A workgroup for each segment of each row; whole rows are reported at once.
template <int DT, int THREADS, bool ENT, bool TOP> __global__ __launch_bounds__(THREADS) void score_rows(ScoreArgs a) {
  __shared__ float lds[THREADS / 64];
  __shared__ typename std::conditional<TOP, Selection, char>::type sel;
  const int64_t row = blockIdx.x / a.split.segs;
  const int seg = blockIdx.x % a.split.segs, lo = seg * a.split.seg;
  const int n = min(a.split.seg, a.in.vocab - lo);
  const auto* p = static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride + lo;
  const float c2 = a.in.scale * kLog2e;
  const RowSums mine = sum_row<DT, THREADS, ENT>(p, n, c2);
  const RowSums r = join_row<THREADS, ENT>(mine, c2, lds);
  if constexpr (TOP) {
    const bool has = static_cast<int>(threadIdx.x) < row_vectors(n, Elem<DT>::N);
    select_top<THREADS>(RowSource<DT, THREADS>{p, n, lo}, has ? order_of(mine.largest) : 0u, a.top, sel);
  }
  if (a.split.segs == 1) {
    if constexpr (TOP) report_row(a, row, r, &sel);
    else report_row(a, row, r, nullptr);
    return;
  }
  Partial* parts = static_cast<Partial*>(a.workspace);
  if (threadIdx.x == 0) parts[blockIdx.x] = {r.largest, r.s, r.t, 0.f};
  if constexpr (TOP) {
    uint64_t* keys = reinterpret_cast<uint64_t*>(parts + a.in.rows * a.split.segs);
    if (static_cast<int>(threadIdx.x) < a.top) keys[static_cast<int64_t>(blockIdx.x) * a.top + threadIdx.x] = sel.top[threadIdx.x];
  }
}

// The sums of a row's segments as the row's, in every thread.
template <int THREADS, bool ENT> __device__ inline RowSums join_parts(const Partial* parts, int segs, float c2, float* lds) {
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
  return join_row<THREADS, ENT>(a, c2, lds);
}

template <int THREADS, bool ENT, bool TOP> __global__ __launch_bounds__(THREADS) void score_join(ScoreArgs a) {
  __shared__ float lds[THREADS / 64];
  __shared__ typename std::conditional<TOP, Selection, char>::type sel;
  const int64_t row = blockIdx.x;
  const int segs = a.split.segs;
  const Partial* parts = static_cast<const Partial*>(a.workspace);
  const RowSums r = join_parts<THREADS, ENT>(parts + row * segs, segs, a.in.scale * kLog2e, lds);
  if constexpr (TOP) {
    const uint64_t* keys = reinterpret_cast<const uint64_t*>(parts + a.in.rows * segs) + row * segs * a.top;
    const KeySource<THREADS> src{keys, segs * a.top};
    uint32_t mine = 0;
    src.each([&](uint32_t order, uint32_t) { mine = max(mine, order); });
    select_top<THREADS>(src, mine, a.top, sel);
    report_row(a, row, r, &sel);
  } else {
    report_row(a, row, r, nullptr);
  }
}

// dz_i = c [ g ([i = t] - p_i) - e p_i (log p_i + H) ] with g, e the gradients of log p_t and H: one
// pass, a workgroup for `span` elements of a row.
template <int DT, bool ENT> __global__ __launch_bounds__(256) void score_grad_rows(ScoreGradArgs a, int spans, int span) {
  constexpr int N = Elem<DT>::N, U = 4, THREADS = 256;
  typedef typename Elem<DT>::T T;
  const int64_t row = blockIdx.x / spans;
  const int lo = static_cast<int>(blockIdx.x % spans) * span, n = min(span, a.in.vocab - lo);
  const T* p = static_cast<const T*>(a.in.z) + row * a.in.stride + lo;
  T* out = static_cast<T*>(a.grad) + row * a.grad_stride + lo;
  const float m = a.norm[2 * row], log_s = a.norm[2 * row + 1], scale = a.in.scale;
  const bool empty = m == -INFINITY && log_s == -INFINITY;
  const int64_t id = load_id(a.targets, row);
  float g = a.grad_logp ? a.grad_logp[row] : 0.f;
  const float e = ENT ? a.grad_entropy[row] : 0.f;
  if (id == a.ignore) g = 0.f;
  else if (id < 0 || id >= a.in.vocab) g = __builtin_nanf("");
  const float at = scale * g, all = scale * (ENT ? g + e * a.entropy[row] : g), each = scale * e;
  const int64_t target = id - lo;
  auto gradient = [&](float z) {
    const float lp = (z - m) * scale - log_s, pr = exp2_hw(lp * kLog2e);
    return ENT ? -pr * (all + each * fmaxf(lp, -200.f)) : -pr * all;
  };
  auto vector = [&](int i, float* z) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = empty ? 0.f : gradient(z[j]);
    const int64_t d = target - static_cast<int64_t>(i) * N;
    if (d >= 0 && d < N && !empty && id != a.ignore) {
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] += j == d ? at : 0.f;
    }
  };
  const int full = n / N, all_vectors = row_vectors(n, N);
  int i = threadIdx.x;
  for (; i + (U - 1) * THREADS < full; i += U * THREADS) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(p + static_cast<int64_t>(i + u * THREADS) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float z[N];
      Elem<DT>::unpack(v[u], z);
      vector(i + u * THREADS, z);
      store16(out + static_cast<int64_t>(i + u * THREADS) * N, Elem<DT>::pack(z));
    }
  }
  for (; i < all_vectors; i += THREADS) {
    float z[N];
    load_vector<DT>(p, i, n, z);
    vector(i, z);
    if (i < full) {
      store16(out + static_cast<int64_t>(i) * N, Elem<DT>::pack(z));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (i * N + j < n) out[i * N + j] = Elem<DT>::put(z[j]);
    }
  }
}

// ---- distillation --------------------------------------------------------------------------------------

struct Teacher {
  int ids[kMaxTeacher];          // -1: no entry
  float q[kMaxTeacher];
};

// The teacher's probabilities of a row into LDS (entries whose id is not a token have none); returns
// sum q (1, or 0 where no entry has any) and, where `largest` is given, the row's loss / T^2:
// sum_k q_k (log q_k - log p_(id_k)).
template <int THREADS> __device__ inline float load_teacher(const DistillArgs& a, int64_t row, Teacher& t, float* lds,
                                                            const RowSums* r, float* kl) {
  const float inv = 1.f / a.temperature;
  float m = -INFINITY;
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const int64_t id = load_id(a.ids, row * a.ids_stride + k);
    const bool named = id >= 0 && id < a.in.vocab;
    const float u = named ? load_as(a.teacher, row * a.teacher_stride + k, a.teacher_dtype) : -INFINITY;
    t.ids[k] = named ? static_cast<int>(id) : -1;
    t.q[k] = u;
    m = u != u ? u : fmaxf(m, u);
  }
  m = block_max<THREADS>(m, lds);
  const float ref = fmaxf(m, kLowest);
  float s = 0.f;
  for (int k = threadIdx.x; k < a.k; k += THREADS)
    if (t.ids[k] >= 0) s += exp2_hw((t.q[k] - ref) * inv * kLog2e);
  s = block_sum<THREADS>(s, lds);
  const float log_s = log2_hw(s) * kLn2;
  const bool none = s == 0.f;
  const bool empty = r && r->s == 0.f;
  const float log_z = r ? log2_hw(r->s) * kLn2 : 0.f;
  float loss = 0.f;
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const float log_q = (t.q[k] - ref) * inv - log_s, q = t.ids[k] >= 0 && !none ? exp2_hw(log_q * kLog2e) : 0.f;
    if (kl && q != 0.f) {
      const float z = load_as(a.in.z, row * a.in.stride + t.ids[k], a.in.dtype);
      loss += q * (log_q - (empty ? -INFINITY : (z - r->m) * a.in.scale - log_z));
    }
    t.q[k] = q;
  }
  if (kl) *kl = block_sum<THREADS>(loss, lds);
  __syncthreads();                        // the entries are there for every thread
  return none ? 0.f : 1.f;
}

// dz_i = w T (Q p_i - sum_{k: id_k = i} q_k) over [lo, lo + n) of a row.  p_i = exp2(c2 (z_i - m) - shift).
// The entries that the teacher names are written again behind the barrier, from the logits themselves.
template <int DT, int THREADS>
__device__ inline void write_gradient(const DistillArgs& a, int64_t row, int lo, int n, float m, float shift, bool empty,
                                      float w, float total, const Teacher& t) {
  constexpr int N = Elem<DT>::N, U = 4;
  typedef typename Elem<DT>::T T;
  const T* p = static_cast<const T*>(a.in.z) + row * a.in.stride + lo;
  T* out = static_cast<T*>(a.grad) + row * a.grad_stride + lo;
  const float c2 = a.in.scale * kLog2e, coef = empty ? 0.f : w * total;
  const float ref = empty ? INFINITY : m;             // every exponential of an empty row is 0
  if (empty) shift = 0.f;
  auto gradient = [&](float z) { return coef * exp2_hw(__builtin_fmaf(z - ref, c2, -shift)); };
  const int full = n / N, all = row_vectors(n, N);
  int i = threadIdx.x;
  for (; i + (U - 1) * THREADS < full; i += U * THREADS) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(p + static_cast<int64_t>(i + u * THREADS) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float z[N];
      Elem<DT>::unpack(v[u], z);
#pragma unroll
      for (int j = 0; j < N; ++j) z[j] = gradient(z[j]);
      store16(out + static_cast<int64_t>(i + u * THREADS) * N, Elem<DT>::pack(z));
    }
  }
  for (; i < all; i += THREADS) {
    float z[N];
    load_vector<DT>(p, i, n, z);
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = gradient(z[j]);
    if (i < full) {
      store16(out + static_cast<int64_t>(i) * N, Elem<DT>::pack(z));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (i * N + j < n) out[i * N + j] = Elem<DT>::put(z[j]);
    }
  }
  __syncthreads();
  if (empty) return;
  for (int k = threadIdx.x; k < a.k; k += THREADS) {
    const int id = t.ids[k], at = id - lo;
    if (id < 0 || at < 0 || at >= n) continue;
    float q = 0.f;
    for (int j = 0; j < a.k; ++j) q += t.ids[j] == id ? t.q[j] : 0.f;      // the same token named twice counts twice
    out[at] = Elem<DT>::put(gradient(Elem<DT>::get(p[at])) - w * q);
  }
}

// A row to a workgroup: its sums, the loss, and with GRAD the gradient from a second reading.
template <int DT, int THREADS, bool GRAD> __global__ __launch_bounds__(THREADS) void distill_rows(DistillArgs a) {
  __shared__ float lds[THREADS / 64];
  __shared__ Teacher teacher;
  const int64_t row = blockIdx.x;
  const auto* p = static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride;
  const float c2 = a.in.scale * kLog2e;
  const RowSums r = join_row<THREADS, false>(sum_row<DT, THREADS, false>(p, a.in.vocab, c2), c2, lds);
  float kl = 0.f;
  const float total = load_teacher<THREADS>(a, row, teacher, lds, &r, &kl);
  if (threadIdx.x == 0) {
    a.loss[row] = kl * a.temperature * a.temperature;
    a.norm[2 * row] = r.largest;
    a.norm[2 * row + 1] = log2_hw(r.s) * kLn2;
  }
  if constexpr (GRAD) {
    const float w = (a.weight ? a.weight[row] : 1.f) * a.temperature;
    write_gradient<DT, THREADS>(a, row, 0, a.in.vocab, r.m, log2_hw(r.s), r.s == 0.f, w, total, teacher);
  }
}

// Few rows: segments' sums, then a workgroup a row joins them and finds the loss.
template <int DT, int THREADS> __global__ __launch_bounds__(THREADS) void distill_parts(DistillArgs a) {
  __shared__ float lds[THREADS / 64];
  const int64_t row = blockIdx.x / a.split.segs;
  const int lo = static_cast<int>(blockIdx.x % a.split.segs) * a.split.seg, n = min(a.split.seg, a.in.vocab - lo);
  const auto* p = static_cast<const typename Elem<DT>::T*>(a.in.z) + row * a.in.stride + lo;
  const float c2 = a.in.scale * kLog2e;
  const RowSums r = join_row<THREADS, false>(sum_row<DT, THREADS, false>(p, n, c2), c2, lds);
  if (threadIdx.x == 0) static_cast<Partial*>(a.workspace)[blockIdx.x] = {r.largest, r.s, 0.f, 0.f};
}
template <int THREADS> __global__ __launch_bounds__(THREADS) void distill_join(DistillArgs a) {
  __shared__ float lds[THREADS / 64];
  __shared__ Teacher teacher;
  const int64_t row = blockIdx.x;
  const RowSums r = join_parts<THREADS, false>(static_cast<const Partial*>(a.workspace) + row * a.split.segs, a.split.segs,
                                               a.in.scale * kLog2e, lds);
  float kl = 0.f;
  load_teacher<THREADS>(a, row, teacher, lds, &r, &kl);
  if (threadIdx.x == 0) {
    a.loss[row] = kl * a.temperature * a.temperature;
    a.norm[2 * row] = r.largest;
    a.norm[2 * row + 1] = log2_hw(r.s) * kLn2;
  }
}

// The gradient from the pair (m, log S) that the loss left, a workgroup for `span` elements of a row.
template <int DT, int THREADS> __global__ __launch_bounds__(THREADS) void distill_grad_rows(DistillArgs a, int spans, int span) {
  __shared__ float lds[THREADS / 64];
  __shared__ Teacher teacher;
  const int64_t row = blockIdx.x / spans;
  const int lo = static_cast<int>(blockIdx.x % spans) * span, n = min(span, a.in.vocab - lo);
  const float total = load_teacher<THREADS>(a, row, teacher, lds, nullptr, nullptr);
  const float m = a.norm[2 * row], log_s = a.norm[2 * row + 1];
  const bool empty = m == -INFINITY && log_s == -INFINITY;
  const float w = (a.weight ? a.weight[row] : 1.f) * a.temperature;
  write_gradient<DT, THREADS>(a, row, lo, n, m, log_s * kLog2e, empty, w, total, teacher);
}

template <class F> hipError_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f(std::integral_constant<int, kF32>{});
    case kBF16: return f(std::integral_constant<int, kBF16>{});
    default: return f(std::integral_constant<int, kF16>{});
  }
}

// `span` elements a workgroup writes of a row, a multiple of a vector; whole rows where that fills
// the device.
void spans_of(int64_t rows, int vocab, int dtype, int compute_units, int* spans, int* span) {
  const RowSplit s = split_rows(rows, vocab, dtype, compute_units);
  *spans = s.segs;
  *span = s.seg;
}

}  // namespace

RowSplit split_rows(int64_t rows, int vocab, int dtype, int compute_units) {
  const int vec = 16 / static_cast<int>(elem_size(dtype));
  const int64_t want = 4 * static_cast<int64_t>(compute_units);
  if (rows >= want) return {1, vocab};
  // at least two rounds of 256 threads for a segment: below that its fixed costs are the larger part
  const int64_t least = 2 * 256 * vec;
  int64_t segs = (want + rows - 1) / rows;
  segs = segs < (vocab + least - 1) / least ? segs : (vocab + least - 1) / least;
  if (segs <= 1) return {1, vocab};
  int64_t seg = (vocab + segs - 1) / segs;
  seg = (seg + vec - 1) / vec * vec;
  segs = (vocab + seg - 1) / seg;
  if (segs <= 1) return {1, vocab};
  return {static_cast<int>(segs), static_cast<int>(seg)};
}

size_t split_workspace(const RowSplit& s, int64_t rows, int top) {
  if (s.segs == 1) return 0;
  return static_cast<size_t>(rows) * static_cast<size_t>(s.segs) * (sizeof(Partial) + sizeof(uint64_t) * static_cast<size_t>(top));
}

hipError_t launch_score(const ScoreArgs& a, hipStream_t stream) {
  constexpr int THREADS = 256;
  const dim3 grid(static_cast<unsigned>(a.in.rows * a.split.segs));
  auto both = [&](auto dt, auto ent, auto top) {
    score_rows<dt.value, THREADS, ent.value, top.value><<<grid, THREADS, 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.split.segs == 1) return e;
    score_join<THREADS, ent.value, top.value><<<dim3(static_cast<unsigned>(a.in.rows)), THREADS, 0, stream>>>(a);
    return hipGetLastError();
  };
  return by_type(a.in.dtype, [&](auto dt) {
    const std::true_type yes;
    const std::false_type no;
    if (a.entropy) return a.top ? both(dt, yes, yes) : both(dt, yes, no);
    return a.top ? both(dt, no, yes) : both(dt, no, no);
  });
}

hipError_t launch_score_grad(const ScoreGradArgs& a, int compute_units, hipStream_t stream) {
  int spans, span;
  spans_of(a.in.rows, a.in.vocab, a.in.dtype, compute_units, &spans, &span);
  const dim3 grid(static_cast<unsigned>(a.in.rows * spans));
  return by_type(a.in.dtype, [&](auto dt) {
    if (a.grad_entropy) score_grad_rows<dt.value, true><<<grid, 256, 0, stream>>>(a, spans, span);
    else score_grad_rows<dt.value, false><<<grid, 256, 0, stream>>>(a, spans, span);
    return hipGetLastError();
  });
}

hipError_t launch_distill_grad(const DistillArgs& a, int compute_units, hipStream_t stream) {
  int spans, span;
  spans_of(a.in.rows, a.in.vocab, a.in.dtype, compute_units, &spans, &span);
  const dim3 grid(static_cast<unsigned>(a.in.rows * spans));
  return by_type(a.in.dtype, [&](auto dt) {
    distill_grad_rows<dt.value, 256><<<grid, 256, 0, stream>>>(a, spans, span);
    return hipGetLastError();
  });
}

hipError_t launch_distill(const DistillArgs& a, int compute_units, hipStream_t stream) {
  constexpr int THREADS = 256;
  return by_type(a.in.dtype, [&](auto dt) {
    const dim3 rows(static_cast<unsigned>(a.in.rows));
    if (a.split.segs == 1) {
      if (a.grad) distill_rows<dt.value, THREADS, true><<<rows, THREADS, 0, stream>>>(a);
      else distill_rows<dt.value, THREADS, false><<<rows, THREADS, 0, stream>>>(a);
      return hipGetLastError();
    }
    distill_parts<dt.value, THREADS><<<dim3(static_cast<unsigned>(a.in.rows * a.split.segs)), THREADS, 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    distill_join<THREADS><<<rows, THREADS, 0, stream>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess || !a.grad) return e;
    return launch_distill_grad(a, compute_units, stream);
  });
}

}  // namespace eh
