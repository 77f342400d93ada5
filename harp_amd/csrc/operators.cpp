// Entry points of the language-model operators (include/eclat_hip.h): everything a kernel assumes
// of its arrays is checked here, on the host, before anything is queued.
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <limits>

#include "handles.hpp"

using namespace eh;

namespace {

constexpr int64_t kMost = int64_t{1} << 46;      // elements of one array, and any stride

size_t size_of(int64_t dtype) {
  switch (dtype) {
    case EH_F32:
    case EH_I32: return 4;
    case EH_BF16:
    case EH_F16: return 2;
    case EH_I64: return 8;
  }
  return 0;
}
bool is_float(int64_t dtype) { return dtype == EH_F32 || dtype == EH_BF16 || dtype == EH_F16; }

bool given(const eh_array& a) { return a.buffer != nullptr || a.offset != 0; }

// An array as the kernels get it: where it starts, and what of memory it covers.
struct Span {
  const char* name = nullptr;
  char* at = nullptr;
  int64_t extent[3] = {1, 1, 1};     // elements along the axes, the last contiguous
  int64_t stride[2] = {0, 0};
  size_t elem = 1;
  bool writes = false;
  bool all = false;                  // a call that finishes has written every element
  HipBuffer* buf = nullptr;
  int64_t last() const { return (extent[0] - 1) * stride[0] + (extent[1] - 1) * stride[1] + extent[2]; }   // elements covered
  int64_t bytes() const { return last() * static_cast<int64_t>(elem); }
  bool dense() const {
    return (extent[1] == 1 || stride[1] == extent[2]) && (extent[0] == 1 || stride[0] == extent[1] * extent[2]);
  }
};

[[noreturn]] void bad(const char* name, const std::string& what) { throw Error(std::string(name) + ": " + what); }

// The call's arrays: collected, checked against each other, their zero fills settled.
class Arrays {
 public:
  explicit Arrays(HipDevice* dev) : dev_(dev) {}

  // `n0` x `n1` x `n2` elements; an absent array gives null unless it is needed.
  void* take(const char* name, const eh_array& a, int64_t n0, int64_t n1, int64_t n2, bool needed, bool writes, bool all = true) {
    if (!given(a)) {
      if (needed) bad(name, "is missing");
      return nullptr;
    }
    Span s;
    s.name = name;
    s.elem = size_of(a.dtype);
    if (!s.elem) bad(name, "unknown element type " + std::to_string(a.dtype));
    s.extent[0] = n0, s.extent[1] = n1, s.extent[2] = n2;
    s.stride[0] = a.stride[0], s.stride[1] = a.stride[1];
    for (int i = 0; i < 2; ++i) {
      if (s.stride[i] < 0 || s.stride[i] > kMost) bad(name, "stride " + std::to_string(s.stride[i]) + " is out of range");
      if (s.extent[i] > 1 && s.stride[i] > 0 && s.extent[i] > kMost / s.stride[i]) bad(name, "is larger than any device memory");
    }
    if (writes) check_apart(s);
    s.writes = writes, s.all = all;
    const bool none = n0 == 0 || n1 == 0 || n2 == 0;
    if (a.buffer) {
      s.buf = &a.buffer->buf;
      if (s.buf->device() != dev_) bad(name, "lives on another device");
      if (!none && (a.offset > s.buf->byte_len() || static_cast<uint64_t>(s.bytes()) > s.buf->byte_len() - a.offset))
        throw Error("Buffer size mismatch: " + std::string(name) + " needs " + std::to_string(s.bytes()) + " bytes behind offset " +
                    std::to_string(a.offset) + ", the buffer has " + std::to_string(s.buf->byte_len()));
      s.at = static_cast<char*>(s.buf->device_ptr()) + a.offset;
    } else {
      if (!none && static_cast<uint64_t>(s.bytes()) > a.bytes)
        throw Error("Buffer size mismatch: " + std::string(name) + " needs " + std::to_string(s.bytes()) + " bytes, has " + std::to_string(a.bytes));
      s.at = reinterpret_cast<char*>(static_cast<uintptr_t>(a.offset));
    }
    if (reinterpret_cast<uintptr_t>(s.at) % s.elem != 0) bad(name, "is not aligned to its elements");
    if (!none) spans_.push_back(s);
    return s.at;
  }
  // A contiguous array of a fixed type.
  template <class T> T* small(const char* name, const eh_array& a, int64_t n, int64_t m, int64_t dtype, bool needed, bool writes, bool all = true) {
    if (given(a) && a.dtype != dtype) bad(name, dtype == EH_F32 ? "has to be f32" : "has to be i32");
    eh_array c = a;
    c.stride[0] = m, c.stride[1] = m;
    return static_cast<T*>(take(name, c, n, 1, m, needed, writes, all));
  }
  void* floats(const char* name, const eh_array& a, int64_t n0, int64_t n1, int64_t n2, int64_t dtype, bool writes, bool all = true) {
    if (given(a) && (!is_float(a.dtype) || (dtype >= 0 && a.dtype != dtype)))
      bad(name, dtype >= 0 ? "has to be of the other arrays' type" : "has to be f32, bf16 or f16");
    return take(name, a, n0, n1, n2, true, writes, all);
  }
  TokenIds ids(const char* name, const eh_array& a, int64_t n, int64_t m) {
    if (given(a) && a.dtype != EH_I32 && a.dtype != EH_I64) bad(name, "has to be i32 or i64");
    return {take(name, a, n, 1, m, true, false), a.dtype == EH_I64};
  }

  // Before the launches: outputs apart from everything else, owed zero fills queued where the call
  // does not overwrite the whole buffer.
  void settle() {
    for (size_t i = 0; i < spans_.size(); ++i)
      for (size_t j = i + 1; j < spans_.size(); ++j)
        if ((spans_[i].writes || spans_[j].writes) && overlap(spans_[i], spans_[j]))
          throw Error(std::string(spans_[i].name) + " and " + spans_[j].name + " overlap in memory, and the call writes one of them");
    for (Span& s : spans_)
      if (s.buf && s.buf->zero_pending() && !overwritten(s)) s.buf->settle();
  }
  // After them.
  void written() {
    for (Span& s : spans_)
      if (s.buf && s.buf->zero_pending()) s.buf->set_zero_pending(false);
  }

 private:
  bool overwritten(const Span& s) const {
    return s.writes && s.all && s.dense() && s.at == s.buf->device_ptr() && static_cast<uint64_t>(s.bytes()) == s.buf->byte_len();
  }
  // An output's elements are all different ones.
  static void check_apart(const Span& s) {
    const int64_t n0 = s.extent[0], n1 = s.extent[1], n2 = s.extent[2], s0 = s.stride[0], s1 = s.stride[1];
    const bool inner = n1 <= 1 || s1 >= n2, outer = n0 <= 1 || s0 >= n2;
    const bool nested = n0 <= 1 || n1 <= 1 || s0 >= (n1 - 1) * s1 + n2 || s1 >= (n0 - 1) * s0 + n2;
    if (!inner || !outer || !nested) bad(s.name, "its rows overlap in memory");
  }
  static bool overlap(const Span& a, const Span& b) {
    const char *a1 = a.at + a.bytes(), *b1 = b.at + b.bytes();
    if (a1 <= b.at || b1 <= a.at) return false;
    // side by side: both walk memory by the same row stride, and neither reaches into the other's columns
    const int64_t ra = row_stride(a), rb = row_stride(b);
    if (ra == 0 || ra != rb) return true;
    const int64_t wa = a.extent[2] * static_cast<int64_t>(a.elem), wb = b.extent[2] * static_cast<int64_t>(b.elem);
    const int64_t d = ((b.at - a.at) % ra + ra) % ra;      // b's columns start d bytes behind a's
    return !(d >= wa && ra - d >= wb);
  }
  // Bytes that every row's start is a multiple of away from the first's; 0: no such grid.
  static int64_t row_stride(const Span& s) {
    int64_t g = 0;
    for (int i = 0; i < 2; ++i)
      if (s.extent[i] > 1) {
        int64_t x = s.stride[i], y = g;
        while (y) {
          const int64_t r = x % y;
          x = y, y = r;
        }
        g = x;
      }
    return g * static_cast<int64_t>(s.elem);
  }

  HipDevice* dev_;
  std::vector<Span> spans_;
};

// The calling thread's current device is the handle's while this lives.
class Current {
 public:
  explicit Current(HipDevice* dev) {
    if (hipGetDevice(&old_) != hipSuccess) old_ = dev->index();
    if (old_ != dev->index()) dev->make_current();
    else old_ = -1;
  }
  ~Current() {
    if (old_ >= 0) (void)hipSetDevice(old_);
  }
  Current(const Current&) = delete;
  Current& operator=(const Current&) = delete;

 private:
  int old_ = -1;
};

// Memory a call works in besides its arrays: the caller's, or a block of the device's pool that goes
// back as soon as the launches are queued (the pool's next owner runs behind them on the stream).
class Workspace {
 public:
  Workspace(HipDevice* dev, Arrays& arrays, const eh_array& a, size_t bytes) : dev_(dev), bytes_(bytes) {
    if (given(a)) {
      eh_array b = a;
      b.dtype = EH_F32;
      const int64_t n = static_cast<int64_t>((bytes + 3) / 4);
      b.stride[0] = b.stride[1] = n;
      at_ = arrays.take("workspace", b, 1, 1, n, false, true, false);
      if (bytes && reinterpret_cast<uintptr_t>(at_) % 16 != 0) bad("workspace", "is not aligned to 16 bytes");
      return;
    }
    if (!bytes) return;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(dev->stream(), &cs) == hipSuccess && cs != hipStreamCaptureStatusNone)
      throw Error("workspace: the call needs " + std::to_string(bytes) + " bytes under stream capture; a graph's replays work in memory that the caller keeps");
    // in powers of two: the pool gives blocks back to requests of their own size
    bytes_ = size_t{1} << 16;
    while (bytes_ < bytes) bytes_ *= 2;
    at_ = dev->allocate(bytes_);
    owned_ = true;
  }
  ~Workspace() {
    if (owned_) dev_->release(at_, bytes_);
  }
  Workspace(const Workspace&) = delete;
  Workspace& operator=(const Workspace&) = delete;
  void* at() const { return at_; }

 private:
  HipDevice* dev_;
  void* at_ = nullptr;
  size_t bytes_;
  bool owned_ = false;
};

void launched(hipError_t e, const char* what) {
  if (e != hipSuccess)
    throw Error(std::string(what) + ": " + hipGetErrorString(e) + " (hip error " + std::to_string(static_cast<int>(e)) + ")");
}

void check_rows(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows > (int64_t{1} << 24)) throw Error("rows: " + std::to_string(rows) + " is out of range (0 to 2^24)");
  if (vocab < 1 || vocab > (int64_t{1} << 30)) throw Error("vocab: " + std::to_string(vocab) + " is out of range (1 to 2^30)");
  // a launch has a workgroup for every 4 KB of a row
  if (rows * ((vocab + 1023) / 1024) >= (int64_t{1} << 31)) throw Error("rows, vocab: " + std::to_string(rows) + " rows of " + std::to_string(vocab) + " are out of range together");
}
float check_scale(double scale, const char* name) {
  const float f = static_cast<float>(scale);
  if (!(scale > 0) || !std::isfinite(f) || f < std::numeric_limits<float>::min() || !std::isfinite(1.f / f) || 1.f / f < std::numeric_limits<float>::min())
    throw Error(std::string(name) + ": has to be a positive finite number");
  return f;
}
void check_sequences(int64_t batch, int64_t time, int64_t width) {
  if (batch < 0 || batch > (int64_t{1} << 22)) throw Error("batch: " + std::to_string(batch) + " is out of range (0 to 2^22)");
  if (time < 0 || time > (int64_t{1} << 31)) throw Error("time: " + std::to_string(time) + " is out of range (0 to 2^31)");
  if (width < 1 || width > (int64_t{1} << 24)) throw Error("width: " + std::to_string(width) + " is out of range (1 to 2^24)");
  if (batch * width > (int64_t{1} << 33)) throw Error("batch, width: " + std::to_string(batch) + " sequences of " + std::to_string(width) + " channels are out of range (2^33 together)");
}

int units(const HipDevice& d) { return std::max(d.profile().compute_units, 1); }

// A launch's threads are counted in 32 bits.
void check_threads(int64_t blocks, int threads, const char* what) {
  if (blocks > ((int64_t{1} << 32) - 1) / threads) throw Error(std::string(what) + ": out of range together, a launch cannot count the threads");
}

RowSplit split_of(const HipDevice& d, int64_t rows, int64_t vocab, const eh_array& logits, bool top) {
  if (!is_float(logits.dtype)) throw Error("logits: has to be f32, bf16 or f16");
  if (rows == 0) return {64, 0, 1, static_cast<int>(vocab)};
  const RowSplit s = split_rows(rows, static_cast<int>(vocab), static_cast<int>(logits.dtype), top, units(d));
  check_threads(rows * s.segs, s.threads, "rows, vocab");
  return s;
}

void check_top(const eh_token_logprobs_args* a) {
  if (a->top < 0 || a->top > kMaxTop || a->top > a->vocab)
    throw Error("top: " + std::to_string(a->top) + " is out of range (0 to " + std::to_string(std::min<int64_t>(kMaxTop, a->vocab)) + ")");
}

LogitRows logit_rows(Arrays& arrays, const eh_array& logits, int64_t rows, int64_t vocab, float scale) {
  LogitRows r{};
  r.z = arrays.floats("logits", logits, rows, 1, vocab, -1, false);
  r.stride = logits.stride[0];
  r.rows = rows;
  r.vocab = static_cast<int>(vocab);
  r.dtype = static_cast<int>(logits.dtype);
  r.scale = scale;
  return r;
}

Sequences sequences(Arrays& arrays, const char* name, const eh_array& a, int64_t batch, int64_t time, int64_t width, int64_t dtype, bool writes, bool all) {
  Sequences s{};
  s.p = arrays.floats(name, a, batch, time, width, dtype, writes, all);
  s.batch = a.stride[0];
  s.step = a.stride[1];
  return s;
}

void check_plan(const ScanArgs& s) {
  const ScanPlan p = plan_scan(s);
  if (p.waves) check_threads(s.batch * p.tiles * p.pieces, 64 * p.waves, "batch, time, width");
}

#define REQUIRE(cond, msg) \
  if (!(cond)) return fail(EH_ERR_INVALID, msg)

}  // namespace

extern "C" {

int eh_token_logprobs_workspace(eh_device* dev, const eh_token_logprobs_args* args, size_t* bytes) {
  REQUIRE(dev && args && bytes, "device, args or bytes is NULL");
  return guard([&] {
    check_rows(args->rows, args->vocab);
    check_top(args);
    *bytes = split_workspace(split_of(dev->dev, args->rows, args->vocab, args->logits, args->top > 0), args->rows, static_cast<int>(args->top));
  });
}

int eh_token_logprobs(eh_device* dev, const eh_token_logprobs_args* args, int sync) {
  REQUIRE(dev && args, "device or args is NULL");
  return guard([&] {
    const eh_token_logprobs_args& a = *args;
    HipDevice* d = &dev->dev;
    check_rows(a.rows, a.vocab);
    check_top(args);
    auto lk = d->stream_lock();
    Current current(d);
    Arrays arrays(d);
    ScoreArgs s{};
    s.split = split_of(*d, a.rows, a.vocab, a.logits, a.top > 0);
    s.in = logit_rows(arrays, a.logits, a.rows, a.vocab, check_scale(a.scale, "scale"));
    s.targets = arrays.ids("targets", a.targets, a.rows, 1);
    if (a.targets.stride[0] != 1 && a.rows > 1) bad("targets", "has to be contiguous");
    s.ignore = a.ignore_index;
    s.logp = arrays.small<float>("logp", a.logp, a.rows, 1, EH_F32, true, true);
    s.entropy = arrays.small<float>("entropy", a.entropy, a.rows, 1, EH_F32, false, true);
    s.norm = arrays.small<float>("norm", a.norm, a.rows, 2, EH_F32, true, true);
    s.top = static_cast<int>(a.top);
    if (a.top) {
      s.top_logp = arrays.small<float>("top_logp", a.top_logp, a.rows, a.top, EH_F32, true, true);
      s.top_ids = arrays.small<int>("top_ids", a.top_ids, a.rows, a.top, EH_I32, true, true);
    }
    Workspace ws(d, arrays, a.workspace, split_workspace(s.split, a.rows, s.top));
    s.workspace = ws.at();
    arrays.settle();
    if (a.rows) launched(launch_score(s, d->stream()), "launch of token_logprobs");
    arrays.written();
    if (sync) d->synchronize();
  });
}

int eh_token_logprobs_backward(eh_device* dev, const eh_token_logprobs_backward_args* args, int sync) {
  REQUIRE(dev && args, "device or args is NULL");
  return guard([&] {
    const eh_token_logprobs_backward_args& a = *args;
    HipDevice* d = &dev->dev;
    check_rows(a.rows, a.vocab);
    auto lk = d->stream_lock();
    Current current(d);
    Arrays arrays(d);
    ScoreGradArgs s{};
    s.in = logit_rows(arrays, a.logits, a.rows, a.vocab, check_scale(a.scale, "scale"));
    s.targets = arrays.ids("targets", a.targets, a.rows, 1);
    if (a.targets.stride[0] != 1 && a.rows > 1) bad("targets", "has to be contiguous");
    s.ignore = a.ignore_index;
    s.norm = arrays.small<const float>("norm", a.norm, a.rows, 2, EH_F32, true, false);
    s.grad_logp = arrays.small<const float>("grad_logp", a.grad_logp, a.rows, 1, EH_F32, false, false);
    s.grad_entropy = arrays.small<const float>("grad_entropy", a.grad_entropy, a.rows, 1, EH_F32, false, false);
    if (s.grad_entropy) s.entropy = arrays.small<const float>("entropy", a.entropy, a.rows, 1, EH_F32, true, false);
    s.grad = arrays.floats("grad", a.grad, a.rows, 1, a.vocab, a.logits.dtype, true);
    s.grad_stride = a.grad.stride[0];
    arrays.settle();
    if (a.rows) launched(launch_score_grad(s, d->stream()), "launch of token_logprobs_backward");
    arrays.written();
    if (sync) d->synchronize();
  });
}

int eh_distill_loss_workspace(eh_device* dev, const eh_distill_loss_args* args, size_t* bytes) {
  REQUIRE(dev && args && bytes, "device, args or bytes is NULL");
  return guard([&] {
    check_rows(args->rows, args->vocab);
    *bytes = split_workspace(split_of(dev->dev, args->rows, args->vocab, args->logits, false), args->rows, 0);
  });
}

static void distill(eh_device* dev, const eh_distill_loss_args& a, bool backward) {
  HipDevice* d = &dev->dev;
  check_rows(a.rows, a.vocab);
  if (a.k < 1 || a.k > kMaxTeacher) throw Error("k: " + std::to_string(a.k) + " is out of range (1 to " + std::to_string(kMaxTeacher) + ")");
  auto lk = d->stream_lock();
  Current current(d);
  Arrays arrays(d);
  DistillArgs s{};
  s.split = split_of(*d, a.rows, a.vocab, a.logits, false);
  s.temperature = check_scale(a.temperature, "temperature");
  s.in = logit_rows(arrays, a.logits, a.rows, a.vocab, 1.f / s.temperature);
  s.teacher = arrays.floats("teacher", a.teacher, a.rows, 1, a.k, -1, false);
  s.teacher_stride = a.teacher.stride[0];
  s.teacher_dtype = static_cast<int>(a.teacher.dtype);
  s.ids = arrays.ids("ids", a.ids, a.rows, a.k);
  s.ids_stride = a.ids.stride[0];
  s.k = static_cast<int>(a.k);
  s.weight = arrays.small<const float>("weight", a.weight, a.rows, 1, EH_F32, false, false);
  s.norm = arrays.small<float>("norm", a.norm, a.rows, 2, EH_F32, true, !backward);
  if (!backward) s.loss = arrays.small<float>("loss", a.loss, a.rows, 1, EH_F32, true, true);
  if (given(a.grad) || backward) {
    s.grad = arrays.floats("grad", a.grad, a.rows, 1, a.vocab, a.logits.dtype, true);
    s.grad_stride = a.grad.stride[0];
  }
  s.held = hold_rows(a.rows, s.in.vocab, s.in.dtype, units(*d));
  if (s.grad) check_threads(a.rows, backward ? 256 : s.held.threads, "rows, vocab");
  const eh_array none{};
  Workspace ws(d, arrays, backward ? none : a.workspace, backward ? 0 : split_workspace(s.split, a.rows, 0));
  s.workspace = ws.at();
  arrays.settle();
  if (a.rows) {
    if (backward) launched(launch_distill_grad(s, d->stream()), "launch of distill_loss_backward");
    else launched(launch_distill(s, d->stream()), "launch of distill_loss");
  }
  arrays.written();
}

int eh_distill_loss(eh_device* dev, const eh_distill_loss_args* args, int sync) {
  REQUIRE(dev && args, "device or args is NULL");
  return guard([&] {
    distill(dev, *args, false);
    if (sync) dev->dev.synchronize();
  });
}

int eh_distill_loss_backward(eh_device* dev, const eh_distill_loss_args* args, int sync) {
  REQUIRE(dev && args, "device or args is NULL");
  return guard([&] {
    distill(dev, *args, true);
    if (sync) dev->dev.synchronize();
  });
}

static ScanArgs scan_sizes(const HipDevice& d, int64_t batch, int64_t time, int64_t width, int64_t log_gate, const eh_array& gate) {
  check_sequences(batch, time, width);
  if (!is_float(gate.dtype)) throw Error("gate: has to be f32, bf16 or f16");
  ScanArgs s{};
  s.compute_units = units(d);
  s.lose_waits = d.lose_waits();
  s.lost = d.lost_wait();
  s.batch = batch, s.time = time, s.width = static_cast<int>(width);
  s.dtype = static_cast<int>(gate.dtype);
  s.log_gate = log_gate != 0;
  const ScanPlan p = plan_scan(s);
  if (p.pieces > (int64_t{1} << 31) / std::max<int64_t>(batch * p.tiles, 1))
    throw Error("batch, time, width: " + std::to_string(batch) + " sequences of " + std::to_string(time) + " steps of " + std::to_string(width) + " channels are out of range together");
  return s;
}

int eh_gated_scan_workspace(eh_device* dev, const eh_gated_scan_args* args, size_t* bytes) {
  REQUIRE(dev && args && bytes, "device, args or bytes is NULL");
  return guard([&] {
    *bytes = scan_workspace(scan_sizes(dev->dev, args->batch, args->time, args->width, args->log_gate, args->gate));
  });
}

int eh_gated_scan_backward_workspace(eh_device* dev, const eh_gated_scan_backward_args* args, size_t* bytes) {
  REQUIRE(dev && args && bytes, "device, args or bytes is NULL");
  return guard([&] {
    *bytes = scan_workspace(scan_sizes(dev->dev, args->batch, args->time, args->width, args->log_gate, args->gate));
  });
}

int eh_gated_scan(eh_device* dev, const eh_gated_scan_args* args, int sync) {
  REQUIRE(dev && args, "device or args is NULL");
  return guard([&] {
    const eh_gated_scan_args& a = *args;
    HipDevice* d = &dev->dev;
    d->check_waits();
    ScanArgs s = scan_sizes(*d, a.batch, a.time, a.width, a.log_gate, a.gate);
    auto lk = d->stream_lock();
    Current current(d);
    Arrays arrays(d);
    const bool all = !given(a.lengths);
    s.gate = sequences(arrays, "gate", a.gate, a.batch, a.time, a.width, -1, false, true);
    s.x = sequences(arrays, "x", a.x, a.batch, a.time, a.width, a.gate.dtype, false, true);
    s.out = sequences(arrays, "out", a.out, a.batch, a.time, a.width, a.gate.dtype, true, all);
    s.state = arrays.small<const float>("state", a.state, a.batch, a.width, EH_F32, false, false);
    s.final_state = arrays.small<float>("final_state", a.final_state, a.batch, a.width, EH_F32, false, true);
    s.lengths = arrays.small<const int>("lengths", a.lengths, a.batch, 1, EH_I32, false, false);
    check_plan(s);
    Workspace ws(d, arrays, a.workspace, scan_board(s, plan_scan(s)));
    s.workspace = ws.at();
    arrays.settle();
    if (a.batch) launched(launch_scan(s, d->stream()), "launch of gated_scan");
    arrays.written();
    if (!sync) return;
    d->synchronize();
    d->check_waits();
  });
}

int eh_gated_scan_backward(eh_device* dev, const eh_gated_scan_backward_args* args, int sync) {
  REQUIRE(dev && args, "device or args is NULL");
  return guard([&] {
    const eh_gated_scan_backward_args& a = *args;
    HipDevice* d = &dev->dev;
    d->check_waits();
    ScanArgs s = scan_sizes(*d, a.batch, a.time, a.width, a.log_gate, a.gate);
    auto lk = d->stream_lock();
    Current current(d);
    Arrays arrays(d);
    const bool all = !given(a.lengths);
    s.gate = sequences(arrays, "gate", a.gate, a.batch, a.time, a.width, -1, false, true);
    s.x = sequences(arrays, "h", a.h, a.batch, a.time, a.width, a.gate.dtype, false, true);
    s.out = sequences(arrays, "grad_h", a.grad_h, a.batch, a.time, a.width, a.gate.dtype, false, true);
    s.grad_gate = sequences(arrays, "grad_gate", a.grad_gate, a.batch, a.time, a.width, a.gate.dtype, true, all);
    s.grad_x = sequences(arrays, "grad_x", a.grad_x, a.batch, a.time, a.width, a.gate.dtype, true, all);
    s.state = arrays.small<const float>("state", a.state, a.batch, a.width, EH_F32, false, false);
    s.grad_final = arrays.small<const float>("grad_final", a.grad_final, a.batch, a.width, EH_F32, false, false);
    s.final_state = arrays.small<float>("grad_state", a.grad_state, a.batch, a.width, EH_F32, false, true);
    s.lengths = arrays.small<const int>("lengths", a.lengths, a.batch, 1, EH_I32, false, false);
    check_plan(s);
    Workspace ws(d, arrays, a.workspace, scan_board(s, plan_scan(s)));
    s.workspace = ws.at();
    arrays.settle();
    if (a.batch) launched(launch_scan_grad(s, d->stream()), "launch of gated_scan_backward");
    arrays.written();
    if (!sync) return;
    d->synchronize();
    d->check_waits();
  });
}

}  // extern "C"
