// The gated linear recurrence h_t = a_t h_(t-1) + x_t over [batch, time, width], and its gradients.
//
// A run of steps maps the state before it to the state behind it, h -> A h + B, and two runs one after
// the other are (A2 A1, A2 B1 + B2).  The backward pass is the same recurrence in reverse order on
// c_t = a_t (g_t + c_(t+1)), what step t hands to step t - 1: its steps are the maps (a_t, a_t g_t), and
//   lambda_t = g_t + c_(t+1),  dx_t = lambda_t,  da_t = lambda_t h_(t-1),  d(log a_t) = da_t a_t,  dh_0 = c_0.
#include "elements.hpp"

namespace eh {
namespace {

constexpr int kSteps = kScanSteps;   // a thread's own steps, held in registers from the only reading

// Where a workgroup leaves what later pieces of the same channels need: 64-bit words (A, B) of its own
// steps, then 32-bit words of the state behind them.  A word says by itself that it is there: nothing
// writes the all-ones pattern that the words start with, which is one of NaN's.
struct Board {
  unsigned int* tickets;         // of each class, kTicketStride words apart
  unsigned long long* maps;
  unsigned int* states;
};
constexpr unsigned int kEmpty = 0xffffffffu;

constexpr int kTicketStride = 8;

// Class `i` of `classes` into which `n` columns are dealt, in runs of neighbours.
struct Class {
  int number;
  int64_t first, columns;
  __device__ Class(int64_t n, int classes, int i) : number(i), first(n / classes * i + min(n % classes, int64_t{i})), columns(n / classes + (i < n % classes)) {}
};

__device__ inline unsigned int word_of(float x) {
  const unsigned int b = __float_as_uint(x);
  return b == kEmpty ? 0x7fc00000u : b;
}

// A word of the board once it is there.  That every wait ends follows from the order of the tickets; one that
// has lasted for half a second all the same (two calls in one workspace at once, say) ends with the
// empty word, which is NaN.
template <class Word> __device__ inline Word wait_for(const Word* p) {
  Word w;
#pragma unroll 1
  for (int left = 1 << 22; (w = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == static_cast<Word>(~0ull) && --left;)
    __builtin_amdgcn_s_sleep(1);
  return w;
}

// A row of at least a vector is read by the vector that ends with it, which `down` channels are moved out of: by
// whole words, then by half a one.  32 bits at a time, since a 64-bit shift whose amount is in the last
// register that a kernel has was seen to take v0's value for it now and then (the gradient of 13 x 1999 x 717
// f16 had about 1000 wrong channels).  What comes in is 0.
template <int DT> __device__ inline u32x4 move_down(u32x4 v, int down) {
  constexpr int N = Elem<DT>::N;
  const int words = N == 4 ? down : down / 2;
  if (words & 2) v = u32x4{v[2], v[3], 0, 0};
  if (words & 1) v = u32x4{v[1], v[2], v[3], 0};
  if (N == 8 && (down & 1)) {
    v = u32x4{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
  }
  return v;
}
// The n < N channels of a row that has no more; what lies behind them is 0.
template <int DT> __device__ inline u32x4 load_few(const typename Elem<DT>::T* p, int n) {
  constexpr int N = Elem<DT>::N;
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= n) break;
    if constexpr (N == 4) v[j] = __float_as_uint(p[j]);
    else v[j / 2] |= static_cast<uint32_t>(p[j]) << (16 * (j % 2));
  }
  return v;
}
// The rows of a piece, from an address that is the same for the whole workgroup; its rows are within
// 4 GiB of it unless FAR, so that an address is one register per thread.
template <int DT, bool FAR> struct PieceRows {
  char* base;
  int64_t step;                  // bytes
  __device__ PieceRows(const Sequences& s, int64_t b, int64_t t, int tile) {
    constexpr int64_t size = sizeof(typename Elem<DT>::T);
    base = static_cast<char*>(s.p) + (b * s.batch + t * s.step + tile) * size;
    step = s.step * size;
  }
  __device__ typename Elem<DT>::T* at(int row, uint32_t channel_bytes) const {
    if constexpr (FAR) return reinterpret_cast<typename Elem<DT>::T*>(base + row * step + channel_bytes);
    else return reinterpret_cast<typename Elem<DT>::T*>(base + (static_cast<uint32_t>(row) * static_cast<uint32_t>(step) + channel_bytes));
  }
};

// kSteps rows from `row` on, each held inside [0, most].  All loads go out together, those of a row's last
// channels too (32 x 512 x 717 f16 16 us and its gradient 23; with those one after the other 21 and 31).
template <int DT, bool FAR> __device__ inline void load_steps(PieceRows<DT, FAR> s, int row, int most, uint32_t cb, int nc, int width, u32x4* v) {
  constexpr int N = Elem<DT>::N;
  if (width >= N) {
    s.base -= 16;                                           // so that offsets stay above 0
    cb += 16 - static_cast<uint32_t>(max(N - nc, 0) * sizeof(typename Elem<DT>::T));
#pragma unroll
    for (int i = 0; i < kSteps; ++i) v[i] = load16(s.at(max(min(row + i, most), 0), cb));
    if (nc < N) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) v[i] = move_down<DT>(v[i], N - width % N);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) v[i] = load_few<DT>(s.at(max(min(row + i, most), 0), cb), nc);
  }
}
template <int DT> __device__ inline void store_channels(typename Elem<DT>::T* p, int n, const float* z) {
  constexpr int N = Elem<DT>::N;
  typedef uint32_t __attribute__((aligned(2))) any32;
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef u32x2 __attribute__((aligned(2))) any64;
  if (n >= N) {
    store16(p, Elem<DT>::pack(z));
    return;
  }
  const u32x4 v = Elem<DT>::pack(z);
  // eight bytes, four, two: whichever n has
  constexpr int half = N / 2;
  uint32_t a = v[0], b = v[1];
  if (n & half) {
    *reinterpret_cast<any64*>(p) = u32x2{a, b};
    p += half, a = v[2], b = v[3];
  }
  if (n & (half / 2)) {
    *reinterpret_cast<any32*>(p) = a;
    p += half / 2, a = b;
  }
  if constexpr (N == 8) {
    if (n & 1) *p = static_cast<uint16_t>(a);
  }
}

// The gates and the added values of a step; behind a sequence's end the step changes nothing.
template <int DT, bool LOG> __device__ inline void step_of(u32x4 vg, u32x4 vx, bool live, float* a, float* x) {
  constexpr int N = Elem<DT>::N;
  Elem<DT>::unpack(vg, a);
  Elem<DT>::unpack(vx, x);
  if (LOG) {
#pragma unroll
    for (int j = 0; j < N; ++j) a[j] = exp2_hw(a[j] * kLog2e);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    a[j] = live ? a[j] : 1.f;
    x[j] = live ? x[j] : 0.f;
  }
}

// A workgroup of W waves has CW channels of W * 512 / LANES steps, its piece: LANES lanes side by side for the
// channels (eight: 128 bytes of a step, a whole cache line), 64 / LANES runs of kSteps steps one after the other in
// each wave, the waves one after the other.  (With eight lanes for rows of fewer vectors most would be idle:
// 256 x 20000 x 9 bf16 278 us instead of 118, 16 x 131072 x 8 f16 96 instead of 38.)  Gates and inputs are read
// once and stay in registers.  Each thread's map, then scans over the lanes, the waves and the pieces of the same
// channels give the state before each thread's steps, and the steps are run from there.
//
// Over the pieces (W == 8; other sequences have one): they form groups of P in the order of the
// steps.  Each leaves its map on the board before it looks at anybody else's, the last of a group the
// state behind it; a piece composes the state before its group with the maps of the group's pieces
// before it, all read at once (128 / LANES pieces: one word a thread in f32, two in 16 bits, where with one
// the wait from group to group made 1 x 131072 x 64 bf16 40 us instead of 29).  Which words are read depends on
// the piece alone, so results do not depend on the order in which workgroups run.
//
// Columns (a sequence's channels of one workgroup's width) are dealt to classes in runs of neighbours;
// a workgroup takes a ticket of its class, of the next one where that has no pieces left.  A class's
// pieces go out in the order of the steps, all of a column's in one class: a piece only waits for
// pieces that have been taken, by workgroups that run, for maps that are left without waiting and for
// the state of the group before, whose waits end for the same reason.  There are as many workgroups as
// pieces, so all are taken.
//
// With eight classes, by the workgroup's number, neighbouring columns are read and written behind one
// L2: where rows do not start at cache lines they share lines, and 13 x 1999 x 717 f16 takes 37 us
// instead of 42 (its gradient 65 instead of 71, 64 x 512 x 1000 f32 87 instead of 107).  Where they do start
// there, one class is better (8 x 4096 x 2048 bf16 89 us instead of 93, the gradient 142 instead of 151).
//
// Bound by memory: 8 x 4096 x 2048 bf16 at 4.6 TB/s forward and 4.7 backward, 1 x 131072 x 512 f32 at 5.4.  Smaller
// pieces read the same at more waits and shares of the board, two vectors a lane do not fit the registers.
template <int DT, int LANES, int W, bool BACK, bool LOG, bool FAR, int EU>
__global__ __launch_bounds__(64 * W, EU) void scan_pieces(ScanArgs a, int pieces, int tiles, int classes, Board board) {
  constexpr int N = Elem<DT>::N, CW = LANES * N, RUN = W * 64 / LANES * kSteps, M = N / 4, P = M * (64 * W / CW);
  static_assert(64 % LANES == 0 && CW <= 64 * W, "a thread for each channel of the workgroup");
  typedef typename Elem<DT>::T T;
  __shared__ float maps[2][W][CW];
  __shared__ float others[2][P][CW];
  __shared__ float before[CW];
  __shared__ int64_t turn[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t columns = a.batch * tiles;
  int64_t column, k = 0;
  if (W == 8 && pieces > 1) {
    if (threadIdx.x == 0) {
      turn[0] = -1;
      for (int i = 0; i < classes; ++i) {
        const Class c(columns, classes, (blockIdx.x + i) % classes);
        if (c.columns == 0) continue;
        const unsigned int t = atomicAdd(board.tickets + c.number * kTicketStride, 1u) + 1u;      // the words start at all ones
        if (t < c.columns * pieces) {
          turn[0] = c.first + t % c.columns;
          turn[1] = t / c.columns;
          break;
        }
      }
    }
    __syncthreads();
    column = turn[0];
    k = turn[1];
    if (column < 0) return;
  } else {
    const Class c(columns, classes, blockIdx.x % classes);
    column = c.first + blockIdx.x / classes;
    if (column >= columns) return;
  }
  if (BACK) k = pieces - 1 - k;
  const int64_t b = column / tiles;
  const int tile = static_cast<int>(column % tiles) * CW;
  const int c0 = tile + (lane % LANES) * N;
  const int nc = a.width - c0;                                            // channels of this thread (above N: N; below 1: none)
  int64_t n = a.time;
  if (a.lengths) n = min(n, max(static_cast<int64_t>(a.lengths[b]), int64_t{0}));
  const int64_t last = n > 0 ? (n - 1) / RUN : 0;                         // the sequence's last piece
  if (k > last) return;
  const int64_t behind = BACK ? last - k : k;                             // pieces before this one, in the order of the steps
  const int run = wave * (64 / LANES) + lane / LANES;                   // this thread's place among the runs
  // counted from the piece's first row: this thread's first row, and how many rows the sequence has from there on
  const int row = (BACK ? W * (64 / LANES) - 1 - run : run) * kSteps, rows = static_cast<int>(min(n - k * RUN, int64_t{RUN}));
  const uint32_t cb = static_cast<uint32_t>((lane % LANES) * N * sizeof(T));

  u32x4 vg[kSteps] = {}, vx[kSteps] = {};
  const bool live = nc > 0 && row < rows;                                 // (runs behind a sequence's end load nothing)
  if (live) {
    load_steps<DT, FAR>({a.gate, b, k * RUN, tile}, row, rows - 1, cb, nc, a.width, vg);
    load_steps<DT, FAR>({BACK ? a.out : a.x, b, k * RUN, tile}, row, rows - 1, cb, nc, a.width, vx);
  }
  // the backward pass: h of the step before each, the rows from the piece before's last on; the first step of all has
  // the state.  Loaded with the rest where a workgroup has the registers, with half of them once the gates are through.
  u32x4 vh[BACK ? kSteps : 1];
  auto load_states = [&] {
    const int first = k > 0 ? 1 : 0;
    if (live) load_steps<DT, FAR>({a.x, b, k * RUN - first, tile}, row - 1 + first, rows - 2 + first, cb, nc, a.width, vh);
  };
  if constexpr (BACK && EU == 2) load_states();
  float A[N], B[N];
#pragma unroll
  for (int j = 0; j < N; ++j) A[j] = 1.f, B[j] = 0.f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = BACK ? kSteps - 1 - s : s;
    float g[N], x[N];
    step_of<DT, LOG>(vg[i], vx[i], row + i < rows, g, x);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      B[j] = BACK ? g[j] * (B[j] + x[j]) : __builtin_fmaf(g[j], B[j], x[j]);
      A[j] *= g[j];
    }
  }
  // the second run over the steps unpacks them again: kept unpacked they would not fit the registers
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    asm volatile("" : "+v"(vg[i]), "+v"(vx[i]));
#pragma unroll
  for (int off = LANES; off < 64; off *= 2) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float pa = __shfl_up(A[j], off), pb = __shfl_up(B[j], off);
      if (lane >= off) {
        B[j] = __builtin_fmaf(A[j], pb, B[j]);
        A[j] *= pa;
      }
    }
  }
  if (lane >= 64 - LANES) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      maps[0][wave][(lane % LANES) * N + j] = A[j];
      maps[1][wave][(lane % LANES) * N + j] = B[j];
    }
  }
  // the map of the runs before this thread's, in its wave
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float pa = __shfl_up(A[j], LANES), pb = __shfl_up(B[j], LANES);
    A[j] = lane < LANES ? 1.f : pa;
    B[j] = lane < LANES ? 0.f : pb;
  }
  __syncthreads();

  // the state before the piece
  const int c = threadIdx.x % CW, p = threadIdx.x / CW, member = static_cast<int>(behind % P);
  const bool mine = tile + c < a.width;
  const float* start = BACK ? a.grad_final : a.state;
  float ma = 1.f, mb = 0.f;                                               // the piece's own map, in the threads with p == 0
  if (p == 0 && mine) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      mb = __builtin_fmaf(maps[0][w][c], mb, maps[1][w][c]);
      ma *= maps[0][w][c];
    }
  }
  const size_t group = static_cast<size_t>(column) * ((pieces + P - 1) / P) + behind / P;
  if (W == 8 && pieces > 1) {
    unsigned long long* words = board.maps + (static_cast<size_t>(column) * pieces + behind) * CW + c;
    if (p == 0 && mine && behind < last && member < P - 1)
      __hip_atomic_store(words, static_cast<unsigned long long>(word_of(ma)) << 32 | word_of(mb), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int q = p + i * (P / M);
      if (!mine || q >= member) break;
      const unsigned long long w = wait_for(words - static_cast<int64_t>(member - q) * CW);
      others[0][q][c] = __uint_as_float(static_cast<unsigned int>(w >> 32));
      others[1][q][c] = __uint_as_float(static_cast<unsigned int>(w));
    }
  }
  if (mine && p == P / M - 1) {
    float h;
    if (behind < P) {
      h = start ? start[b * a.width + tile + c] : 0.f;
    } else {
      h = __uint_as_float(wait_for(board.states + (group - 1) * CW + c));
    }
    before[c] = h;
  }
  __syncthreads();
  if (p == 0 && mine) {
    float h = before[c];
    for (int i = 0; i < member; ++i) h = __builtin_fmaf(others[0][i][c], h, others[1][i][c]);
    before[c] = h;
    const float next = __builtin_fmaf(ma, h, mb);
    if (behind == last) {
      if (a.final_state) a.final_state[b * a.width + tile + c] = next;
    } else if (member == P - 1) {
      __hip_atomic_store(board.states + group * CW + c, word_of(next), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // NaN of its own, or a wait that gave up: the host is told.  (The state is looked up again; to keep its word from
    // the first look would delay every piece, 1 x 131072 x 64 bf16 by 0.6 us of 29.)
    if (W == 8 && pieces > 1 && next != next) {
      bool lost = behind >= P && __hip_atomic_load(board.states + (group - 1) * CW + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == kEmpty;
#pragma unroll 1
      for (int i = 0; i < member; ++i) lost |= __float_as_uint(others[0][i][c]) == kEmpty;
      if (lost) __hip_atomic_store(a.lost, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
  }
  __syncthreads();
  if (nc <= 0) return;
  float h[N];
#pragma unroll
  for (int j = 0; j < N; ++j) h[j] = before[(lane % LANES) * N + j];
  for (int w = 0; w < wave; ++w)
#pragma unroll
    for (int j = 0; j < N; ++j) h[j] = __builtin_fmaf(maps[0][w][(lane % LANES) * N + j], h[j], maps[1][w][(lane % LANES) * N + j]);
#pragma unroll
  for (int j = 0; j < N; ++j) h[j] = __builtin_fmaf(A[j], h[j], B[j]);

  if constexpr (!BACK) {
    const PieceRows<DT, FAR> out(a.out, b, k * RUN, tile);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float g[N], x[N];
      step_of<DT, LOG>(vg[i], vx[i], true, g, x);
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = __builtin_fmaf(g[j], h[j], x[j]);
      if (row + i < rows) store_channels<DT>(out.at(row + i, cb), nc, h);
    }
  } else {
    const PieceRows<DT, FAR> dg(a.grad_gate, b, k * RUN, tile), dx(a.grad_x, b, k * RUN, tile);
    if constexpr (EU != 2) load_states();
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      if (row + i >= rows) continue;                                       // h stays what came from behind
      float g[N], x[N], prev[N];
      step_of<DT, LOG>(vg[i], vx[i], true, g, x);
      Elem<DT>::unpack(vh[i], prev);
      if (i == 0 && row == 0 && k == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) prev[j] = a.state && j < nc ? a.state[b * a.width + c0 + j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x[j] += h[j];                                                     // lambda
        prev[j] *= x[j];
        if (LOG) prev[j] *= g[j];
        h[j] = g[j] * x[j];
      }
      store_channels<DT>(dx.at(row + i, cb), nc, x);
      store_channels<DT>(dg.at(row + i, cb), nc, prev);
    }
  }
}

// One channel of a short sequence, step by step.
template <int DT, bool BACK, bool LOG> __device__ inline void scan_channel(const ScanArgs& a, int64_t b, int c, int n) {
  typedef typename Elem<DT>::T T;
  auto at = [&](const Sequences& s, int t) { return static_cast<T*>(s.p) + b * s.batch + t * s.step + c; };
  const int64_t end = b * a.width + c;
  const float* start = BACK ? a.grad_final : a.state;
  float h = start ? start[end] : 0.f;
  for (int s = 0; s < n; ++s) {
    const int t = BACK ? n - 1 - s : s;
    float g = Elem<DT>::get(*at(a.gate, t));
    if (LOG) g = exp2_hw(g * kLog2e);
    if constexpr (!BACK) {
      h = __builtin_fmaf(g, h, Elem<DT>::get(*at(a.x, t)));
      *at(a.out, t) = Elem<DT>::put(h);
    } else {
      const float l = Elem<DT>::get(*at(a.out, t)) + h;
      const float prev = (t > 0 ? Elem<DT>::get(*at(a.x, t - 1)) : a.state ? a.state[end] : 0.f) * l;
      *at(a.grad_x, t) = Elem<DT>::put(l);
      *at(a.grad_gate, t) = Elem<DT>::put(LOG ? prev * g : prev);
      h = g * l;
    }
  }
  if (a.final_state) a.final_state[end] = h;
}

// Short sequences (a decoding step: STEPS = 1), a thread for a vector of channels: the loads of STEPS
// steps first, then the steps.
template <int DT, int STEPS, bool BACK, bool LOG> __global__ __launch_bounds__(256, BACK ? 3 : 4) void scan_short(ScanArgs a, int vectors) {
  constexpr int N = Elem<DT>::N;
  typedef typename Elem<DT>::T T;
  const int64_t i = blockIdx.x * int64_t{256} + threadIdx.x, b = i / vectors;
  if (b >= a.batch) return;
  const int c0 = static_cast<int>(i % vectors) * N;
  int n = static_cast<int>(a.time);
  if (a.lengths) n = min(n, max(a.lengths[b], 0));
  if (a.width - c0 < N) {
    for (int c = c0; c < a.width; ++c) scan_channel<DT, BACK, LOG>(a, b, c, n);
    return;
  }
  auto row = [&](const Sequences& s, int t) { return static_cast<T*>(s.p) + b * s.batch + t * s.step + c0; };
  const int64_t end = b * a.width + c0;
  auto get = [&](const float* p, float* z) {
#pragma unroll
    for (int j = 0; j < N; j += 4) Elem<kF32>::unpack(p ? load16(p + end + j) : u32x4{0, 0, 0, 0}, z + j);
  };
  float h[N], first[N];
  get(BACK ? a.grad_final : a.state, h);
  if (BACK) get(a.state, first);
  const int parts = (n + STEPS - 1) / STEPS;
  for (int part = 0; part < parts; ++part) {
    const int t0 = (BACK ? parts - 1 - part : part) * STEPS;
    u32x4 vg[STEPS] = {}, vx[STEPS] = {}, vh[STEPS] = {};
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (t0 + i < n) {
        vg[i] = load16(row(a.gate, t0 + i));
        vx[i] = load16(row(BACK ? a.out : a.x, t0 + i));
        if (BACK && t0 + i > 0) vh[i] = load16(row(a.x, t0 + i - 1));
      }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = BACK ? STEPS - 1 - s : s, t = t0 + i;
      if (t >= n) continue;
      float g[N], x[N];
      step_of<DT, LOG>(vg[i], vx[i], true, g, x);
      if constexpr (!BACK) {
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = __builtin_fmaf(g[j], h[j], x[j]);
        store16(row(a.out, t), Elem<DT>::pack(h));
      } else {
        float prev[N];
        Elem<DT>::unpack(vh[i], prev);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (t == 0) prev[j] = first[j];
          x[j] += h[j];
          prev[j] *= x[j];
          if (LOG) prev[j] *= g[j];
          h[j] = g[j] * x[j];
        }
        store16(row(a.grad_x, t), Elem<DT>::pack(x));
        store16(row(a.grad_gate, t), Elem<DT>::pack(prev));
      }
    }
  }
  if (!a.final_state) return;
#pragma unroll
  for (int j = 0; j < N; j += 4) store16(a.final_state + end + j, Elem<kF32>::pack(h + j));
}

// For tests of what a lost wait leads to: every column's first turn is taken, by nobody.
__global__ __launch_bounds__(64) void skip_turns(unsigned int* tickets, int64_t columns, int classes) {
  if (static_cast<int>(threadIdx.x) < classes) tickets[threadIdx.x * kTicketStride] = static_cast<unsigned int>(Class(columns, classes, threadIdx.x).columns) - 1u;
}

__global__ __launch_bounds__(256) void clear_board(unsigned int* p, size_t n) {
  for (size_t i = blockIdx.x * size_t{256} + threadIdx.x; i < n; i += size_t{256} * gridDim.x) p[i] = kEmpty;
}

template <class F> hipError_t by_type(int dtype, F&& f) {
  switch (dtype) {
    case kF32: return f(std::integral_constant<int, kF32>{});
    case kBF16: return f(std::integral_constant<int, kBF16>{});
    default: return f(std::integral_constant<int, kF16>{});
  }
}

template <int N> using Int = std::integral_constant<int, N>;

template <bool BACK> hipError_t launch(const ScanArgs& a, hipStream_t stream) {
  const ScanPlan p = plan_scan(a);
  if (p.waves == 0) {
    return by_type(a.dtype, [&](auto dt) {
      const int vectors = (a.width + Elem<dt.value>::N - 1) / Elem<dt.value>::N;
      const unsigned grid = static_cast<unsigned>((a.batch * vectors + 255) / 256);
      auto go = [&](auto steps) {
        return a.log_gate ? queue(scan_short<dt.value, steps.value, BACK, true>, grid, 256, 0, stream, a, vectors)
                          : queue(scan_short<dt.value, steps.value, BACK, false>, grid, 256, 0, stream, a, vectors);
      };
      if (a.time <= 1) return go(Int<1>{});
      return go(Int<kSteps>{});
    });
  }
  Board board{};
  if (p.pieces > 1) {
    const size_t words = scan_board(a, p) / 4;
    board.tickets = static_cast<unsigned int*>(a.workspace);
    board.maps = reinterpret_cast<unsigned long long*>(board.tickets + kTicketBytes / 4);
    board.states = reinterpret_cast<unsigned int*>(board.maps + a.batch * p.tiles * p.pieces * p.channels);
    const size_t blocks = (words + 1023) / 1024;
    if (hipError_t e = queue(clear_board, static_cast<unsigned>(blocks < 1024 ? blocks : 1024), 256, 0, stream, board.tickets, words)) return e;
    if (a.lose_waits)
      if (hipError_t e = queue(skip_turns, 1, 64, 0, stream, board.tickets, a.batch * p.tiles, p.classes)) return e;
  }
  const unsigned grid = static_cast<unsigned>(a.batch * p.tiles * p.pieces);
  return by_type(a.dtype, [&](auto dt) {
    auto go = [&](auto lanes, auto waves, auto is_far, auto eu) {
      const int pieces = static_cast<int>(p.pieces), tiles = static_cast<int>(p.tiles);
      return a.log_gate ? queue(scan_pieces<dt.value, lanes.value, waves.value, BACK, true, is_far.value, eu.value>, grid, 64 * waves.value, 0, stream, a, pieces, tiles, p.classes, board)
                        : queue(scan_pieces<dt.value, lanes.value, waves.value, BACK, false, is_far.value, eu.value>, grid, 64 * waves.value, 0, stream, a, pieces, tiles, p.classes, board);
    };
    const std::false_type near;
    if (p.far) return go(Int<8>{}, Int<8>{}, std::true_type{}, Int<2>{});
    if (p.lanes == 2) return p.waves == 1 ? go(Int<2>{}, Int<1>{}, near, Int<2>{}) : go(Int<2>{}, Int<8>{}, near, Int<4>{});
    if (p.lanes == 4) return p.waves == 1 ? go(Int<4>{}, Int<1>{}, near, Int<2>{}) : go(Int<4>{}, Int<8>{}, near, Int<4>{});
    if (p.waves == 1) return go(Int<8>{}, Int<1>{}, near, Int<2>{});
    if (p.waves == 2) return go(Int<8>{}, Int<2>{}, near, Int<2>{});
    if (p.waves == 4) return go(Int<8>{}, Int<4>{}, near, Int<2>{});
    if (p.waves == 16) return go(Int<8>{}, Int<16>{}, near, Int<4>{});
    if constexpr (BACK && dt.value != kF32) {
      if (p.wide) return go(Int<8>{}, Int<8>{}, near, Int<2>{});
    }
    return go(Int<8>{}, Int<8>{}, near, Int<4>{});
  });
}

}  // namespace

hipError_t launch_scan(const ScanArgs& a, hipStream_t stream) { return launch<false>(a, stream); }
hipError_t launch_scan_grad(const ScanArgs& a, hipStream_t stream) { return launch<true>(a, stream); }

}  // namespace eh
