// The operators' entry points without a GPU: their checks of arguments, and the plans their launches
// go by.  The device, its buffers and the launches are stand-ins; a launch touches the first and the
// last element of every array it was given (built with AddressSanitizer), so an array that the checks
// let through too small ends the program.
#include "../harp_amd/csrc/operators.cpp"

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

static std::string g_error;
static int g_launches = 0, g_fills = 0, g_syncs = 0, g_allocations = 0, g_freed = 0;
static bool g_capturing = false, g_launch_fails = false;

// ---- stand-ins ---------------------------------------------------------------------------------------
namespace eh {
int fail(int code, const std::string& m) {
  g_error = m;
  return code;
}
int classify(const std::string& m) {
  if (m.find("Buffer size mismatch") != std::string::npos) return EH_ERR_SIZE;
  if (m.find("hip error") != std::string::npos) return EH_ERR_DEVICE;
  return EH_ERR_INVALID;
}
HipDevice::HipDevice(int index) : index_(index) { profile_.compute_units = 256; }
HipDevice::HipDevice(int index, hipStream_t s) : index_(index), stream_(s) { profile_.compute_units = 256; }
HipDevice::~HipDevice() {}
void HipDevice::make_current() const {}
void HipDevice::synchronize() const { ++g_syncs; }
void* HipDevice::allocate(size_t n) {
  ++g_allocations;
  return std::malloc(n);
}
void HipDevice::release(void* p, size_t) {
  ++g_freed;
  std::free(p);
}
HipBuffer::HipBuffer(HipDevice* d, size_t n) : dev_(d), bytes_(n) {
  ptr_ = std::malloc(n ? n : 1);
  zero_pending_ = true;
}
HipBuffer::~HipBuffer() { std::free(ptr_); }
void HipBuffer::settle() {
  if (zero_pending_) ++g_fills, std::memset(ptr_, 0, bytes_);
  zero_pending_ = false;
}

static volatile char g_sink;
static void touch(const void* p, int64_t n, size_t size, bool write = false) {
  if (!p || n <= 0) return;
  char* b = static_cast<char*>(const_cast<void*>(p));
  if (write) b[0] = 1, b[n * static_cast<int64_t>(size) - 1] = 1;
  g_sink = static_cast<char>(b[0] + b[n * static_cast<int64_t>(size) - 1]);
}
static void touch_rows(const void* p, int64_t rows, int64_t stride, int64_t n, size_t size, bool write = false) {
  if (p && rows > 0) touch(p, n, size, write), touch(static_cast<const char*>(p) + (rows - 1) * stride * static_cast<int64_t>(size), n, size, write);
}
static hipError_t done() {
  ++g_launches;
  return g_launch_fails ? hipErrorLaunchFailure : hipSuccess;
}
hipError_t launch_score(const ScoreArgs& a, hipStream_t) {
  touch_rows(a.in.z, a.in.rows, a.in.stride, a.in.vocab, elem_size(a.in.dtype));
  touch(a.targets.ids, a.in.rows, a.targets.wide ? 8 : 4);
  touch(a.logp, a.in.rows, 4, true), touch(a.entropy, a.in.rows, 4, true), touch(a.norm, 2 * a.in.rows, 4, true);
  touch(a.top_logp, a.in.rows * a.top, 4, true), touch(a.top_ids, a.in.rows * a.top, 4, true);
  touch(a.workspace, static_cast<int64_t>(split_workspace(a.split, a.in.rows, a.top)), 1, true);
  return done();
}
hipError_t launch_score_grad(const ScoreGradArgs& a, hipStream_t) {
  touch_rows(a.in.z, a.in.rows, a.in.stride, a.in.vocab, elem_size(a.in.dtype));
  touch(a.targets.ids, a.in.rows, a.targets.wide ? 8 : 4);
  touch(a.norm, 2 * a.in.rows, 4), touch(a.entropy, a.in.rows, 4), touch(a.grad_logp, a.in.rows, 4), touch(a.grad_entropy, a.in.rows, 4);
  touch_rows(a.grad, a.in.rows, a.grad_stride, a.in.vocab, elem_size(a.in.dtype), true);
  return done();
}
static void touch_distill(const DistillArgs& a) {
  touch_rows(a.in.z, a.in.rows, a.in.stride, a.in.vocab, elem_size(a.in.dtype));
  touch_rows(a.teacher, a.in.rows, a.teacher_stride, a.k, elem_size(a.teacher_dtype));
  touch_rows(a.ids.ids, a.in.rows, a.ids_stride, a.k, a.ids.wide ? 8 : 4);
  touch(a.weight, a.in.rows, 4), touch(a.norm, 2 * a.in.rows, 4);
  touch_rows(a.grad, a.in.rows, a.grad_stride, a.in.vocab, elem_size(a.in.dtype), true);
}
hipError_t launch_distill(const DistillArgs& a, hipStream_t) {
  touch_distill(a);
  touch(a.loss, a.in.rows, 4, true);
  touch(a.workspace, static_cast<int64_t>(split_workspace(a.split, a.in.rows, 0)), 1, true);
  return done();
}
hipError_t launch_distill_grad(const DistillArgs& a, hipStream_t) {
  touch_distill(a);
  return done();
}
static void touch_sequences(const Sequences& s, const ScanArgs& a, bool write) {
  if (!s.p || a.time == 0) return;
  for (int64_t b : {int64_t{0}, a.batch - 1})
    touch_rows(static_cast<char*>(s.p) + b * s.batch * static_cast<int64_t>(elem_size(a.dtype)), a.time, s.step, a.width, elem_size(a.dtype), write);
}
static hipError_t scan(const ScanArgs& a, bool back) {
  touch_sequences(a.gate, a, false), touch_sequences(a.x, a, false), touch_sequences(a.out, a, !back);
  touch_sequences(a.grad_gate, a, true), touch_sequences(a.grad_x, a, true);
  const int64_t n = a.batch * a.width;
  touch(a.state, n, 4), touch(a.final_state, n, 4, true), touch(a.grad_final, n, 4), touch(a.lengths, a.batch, 4);
  touch(a.workspace, static_cast<int64_t>(scan_workspace(a)), 1, true);
  return done();
}
hipError_t launch_scan(const ScanArgs& a, hipStream_t) { return scan(a, false); }
hipError_t launch_scan_grad(const ScanArgs& a, hipStream_t) { return scan(a, true); }
}  // namespace eh

extern "C" {
hipError_t hipGetDevice(int* d) {
  *d = 0;
  return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
}

// ---- the tests ---------------------------------------------------------------------------------------

static int g_failures = 0, g_checks = 0;
#define CHECK(cond)                                                             \
  do {                                                                          \
    ++g_checks;                                                                 \
    if (!(cond)) {                                                              \
      ++g_failures;                                                             \
      std::printf("%s:%d: %s (%s)\n", __FILE__, __LINE__, #cond, g_error.c_str()); \
    }                                                                           \
  } while (0)

static bool refused(int code, int want, const char* word) { return code == want && g_error.find(word) != std::string::npos; }

struct Pool {
  std::vector<eh_buffer*> all;
  eh_device* dev;
  explicit Pool(eh_device* d) : dev(d) {}
  ~Pool() {
    for (eh_buffer* b : all) delete b;
  }
  eh_array array(int64_t n0, int64_t n1, int64_t n2, int dtype, int64_t more = 0) {
    const size_t size = size_of(dtype);
    eh_buffer* b = new eh_buffer(&dev->dev, static_cast<size_t>(n0 * n1 * n2 + more) * size);
    all.push_back(b);
    eh_array a{};
    a.buffer = b;
    a.stride[0] = n1 * n2, a.stride[1] = n2, a.dtype = dtype;
    return a;
  }
  eh_array outside(const eh_array& a) {        // the same memory as the caller's own
    eh_array r = a;
    r.bytes = a.buffer->buf.byte_len();
    r.offset = reinterpret_cast<uint64_t>(a.buffer->buf.device_ptr());
    r.buffer = nullptr;
    return r;
  }
};

static eh_token_logprobs_args score_args(Pool& p, int64_t n, int64_t v, int64_t top, int dtype = EH_F32) {
  eh_token_logprobs_args a{};
  a.rows = n, a.vocab = v, a.top = top, a.ignore_index = -1, a.scale = 1.0;
  a.logits = p.array(n, 1, v, dtype);
  a.targets = p.array(n, 1, 1, EH_I64);
  a.logp = p.array(n, 1, 1, EH_F32), a.entropy = p.array(n, 1, 1, EH_F32), a.norm = p.array(n, 1, 2, EH_F32);
  if (top) a.top_logp = p.array(n, 1, top, EH_F32), a.top_ids = p.array(n, 1, top, EH_I32);
  return a;
}

static void scores(eh_device* d, eh_device* other) {
  Pool p(d), q(other);
  const eh_token_logprobs_args ok = score_args(p, 6, 50, 4);
  CHECK(eh_token_logprobs(d, &ok, 0) == EH_OK);
  CHECK(g_fills == 2);                           // logits and targets: what the call writes needs no zeros
  for (eh_array eh_token_logprobs_args::*m : {&eh_token_logprobs_args::logits, &eh_token_logprobs_args::targets, &eh_token_logprobs_args::logp,
                                              &eh_token_logprobs_args::entropy, &eh_token_logprobs_args::norm, &eh_token_logprobs_args::top_logp,
                                              &eh_token_logprobs_args::top_ids}) {
    eh_token_logprobs_args a = ok;
    (a.*m) = p.outside(ok.*m);
    CHECK(eh_token_logprobs(d, &a, 0) == EH_OK);
    (a.*m).bytes -= 1;
    CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_SIZE, "size mismatch"));
    a = ok;
    (a.*m).offset = size_of((a.*m).dtype);
    CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_SIZE, "size mismatch"));
    (a.*m).offset = ~uint64_t{0} - 3;
    CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_SIZE, "size mismatch"));
    (a.*m).offset = 1;
    CHECK(eh_token_logprobs(d, &a, 0) != EH_OK);
    a = ok;
    (a.*m) = eh_array{};
    CHECK(m == &eh_token_logprobs_args::entropy ? eh_token_logprobs(d, &a, 0) == EH_OK : refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, ""));
    a = ok;
    (a.*m).dtype = 77;
    CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, ""));
    a = ok;
    (a.*m) = q.array(6, 1, 50, static_cast<int>((a.*m).dtype));
    CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, "another device"));
  }
  auto bad = [&](auto change, const char* word) {
    eh_token_logprobs_args a = ok;
    change(a);
    const int before = g_launches;
    CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, word));
    CHECK(g_launches == before);
  };
  bad([](auto& a) { a.rows = -1; }, "rows");
  bad([](auto& a) { a.rows = int64_t{1} << 40; }, "rows");
  bad([](auto& a) { a.vocab = 0; }, "vocab");
  bad([](auto& a) { a.vocab = int64_t{1} << 31; }, "vocab");
  bad([](auto& a) { a.rows = 1 << 24, a.vocab = 1 << 30; }, "out of range together");
  bad([](auto& a) { a.rows = 1 << 23, a.vocab = 1 << 17; }, "out of range together");
  bad([](auto& a) { a.top = -1; }, "top");
  bad([](auto& a) { a.top = 33; }, "top");
  bad([](auto& a) { a.vocab = 3; }, "top");
  bad([](auto& a) { a.scale = 0; }, "scale");
  bad([](auto& a) { a.scale = -1; }, "scale");
  bad([](auto& a) { a.scale = 1e-45; }, "scale");
  bad([](auto& a) { a.scale = 1e39; }, "scale");
  bad([](auto& a) { a.scale = std::nan(""); }, "scale");
  bad([](auto& a) { a.logits.stride[0] = -50; }, "stride");
  bad([](auto& a) { a.logits.stride[0] = int64_t{1} << 60; }, "stride");
  bad([](auto& a) { a.logits.stride[0] = int64_t{1} << 45; }, "larger");
  bad([](auto& a) { a.logits.dtype = EH_I32; }, "f32, bf16 or f16");
  bad([](auto& a) { a.targets.dtype = EH_F32; }, "i32 or i64");
  bad([](auto& a) { a.targets.stride[0] = 0; }, "contiguous");
  bad([](auto& a) { a.top_ids.dtype = EH_I64; }, "i32");
  bad([](auto& a) { a.logp.dtype = EH_BF16; }, "f32");
  bad([](auto& a) { a.logp = a.entropy; }, "overlap");
  bad([](auto& a) { a.logp = a.logits, a.logp.dtype = EH_F32; }, "overlap");
  CHECK(eh_token_logprobs(nullptr, &ok, 0) == EH_ERR_INVALID && eh_token_logprobs(d, nullptr, 0) == EH_ERR_INVALID);
  eh_token_logprobs_args a = ok;
  a.logits.stride[0] = 0;                        // one row of logits for all: fine to read
  CHECK(eh_token_logprobs(d, &a, 1) == EH_OK && g_syncs == 1);
  a = ok;
  a.rows = 0;
  const int before = g_launches;
  CHECK(eh_token_logprobs(d, &a, 0) == EH_OK && g_launches == before);
  g_launch_fails = true;
  CHECK(refused(eh_token_logprobs(d, &ok, 0), EH_ERR_DEVICE, "hip error"));
  g_launch_fails = false;
}

static void workspaces(eh_device* d) {
  Pool p(d);
  eh_token_logprobs_args a = score_args(p, 2, 300000, 20);
  size_t n = 0;
  CHECK(eh_token_logprobs_workspace(d, &a, &n) == EH_OK && n > 0);
  const int before = g_allocations;
  CHECK(eh_token_logprobs(d, &a, 0) == EH_OK && g_allocations == before + 1 && g_freed == g_allocations);
  g_capturing = true;
  CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, "workspace"));
  a.workspace = p.array(1, 1, static_cast<int64_t>(n + 3) / 4, EH_F32);
  CHECK(eh_token_logprobs(d, &a, 0) == EH_OK && g_allocations == before + 1);
  a.workspace = p.array(1, 1, static_cast<int64_t>(n) / 4 - 1, EH_F32);
  CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_SIZE, "workspace"));
  a.workspace = p.array(1, 1, static_cast<int64_t>(n), EH_F32);
  a.workspace.offset = 4;
  CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, "16 bytes"));
  a.workspace = a.logits;
  CHECK(refused(eh_token_logprobs(d, &a, 0), EH_ERR_INVALID, "overlap"));
  g_capturing = false;
}

static void gradients(eh_device* d) {
  Pool p(d);
  eh_token_logprobs_backward_args ok{};
  ok.rows = 5, ok.vocab = 40, ok.ignore_index = -1, ok.scale = 0.5;
  ok.logits = p.array(5, 1, 40, EH_F16), ok.grad = p.array(5, 1, 40, EH_F16), ok.targets = p.array(5, 1, 1, EH_I32);
  ok.norm = p.array(5, 1, 2, EH_F32), ok.entropy = p.array(5, 1, 1, EH_F32), ok.grad_logp = p.array(5, 1, 1, EH_F32);
  ok.grad_entropy = p.array(5, 1, 1, EH_F32);
  CHECK(eh_token_logprobs_backward(d, &ok, 0) == EH_OK);
  auto bad = [&](auto change, int code, const char* word) {
    eh_token_logprobs_backward_args a = ok;
    change(a);
    CHECK(refused(eh_token_logprobs_backward(d, &a, 0), code, word));
  };
  bad([](auto& a) { a.entropy = eh_array{}; }, EH_ERR_INVALID, "entropy");
  bad([](auto& a) { a.norm = eh_array{}; }, EH_ERR_INVALID, "norm");
  bad([](auto& a) { a.grad = a.logits; }, EH_ERR_INVALID, "overlap");
  bad([](auto& a) { a.grad.dtype = EH_BF16; }, EH_ERR_INVALID, "other arrays' type");
  bad([](auto& a) { a.grad.stride[0] = 39; }, EH_ERR_INVALID, "rows overlap");
  bad([](auto& a) { a.grad.stride[0] = 0; }, EH_ERR_INVALID, "rows overlap");
  bad([](auto& a) { a.grad.stride[0] = 41; }, EH_ERR_SIZE, "size mismatch");
  eh_token_logprobs_backward_args a = ok;
  a.grad_logp = a.grad_entropy = a.entropy = eh_array{};
  CHECK(eh_token_logprobs_backward(d, &a, 0) == EH_OK);
  // logits and gradient side by side in the rows of one buffer
  a = ok;
  a.logits = p.array(5, 1, 80, EH_F16), a.grad = a.logits;
  a.grad.offset = 80;
  CHECK(eh_token_logprobs_backward(d, &a, 0) == EH_OK);
  a.grad.offset = 78;
  CHECK(refused(eh_token_logprobs_backward(d, &a, 0), EH_ERR_INVALID, "overlap"));
}

static void distillation(eh_device* d) {
  Pool p(d);
  eh_distill_loss_args ok{};
  ok.rows = 4, ok.vocab = 30, ok.k = 5, ok.temperature = 2.0;
  ok.logits = p.array(4, 1, 30, EH_BF16), ok.teacher = p.array(4, 1, 5, EH_F32), ok.ids = p.array(4, 1, 5, EH_I32);
  ok.weight = p.array(4, 1, 1, EH_F32), ok.loss = p.array(4, 1, 1, EH_F32), ok.norm = p.array(4, 1, 2, EH_F32), ok.grad = p.array(4, 1, 30, EH_BF16);
  CHECK(eh_distill_loss(d, &ok, 0) == EH_OK && eh_distill_loss_backward(d, &ok, 0) == EH_OK);
  for (int backward = 0; backward < 2; ++backward) {
    auto call = [&](const eh_distill_loss_args& a) { return backward ? eh_distill_loss_backward(d, &a, 0) : eh_distill_loss(d, &a, 0); };
    auto bad = [&](auto change, int code, const char* word) {
      eh_distill_loss_args a = ok;
      change(a);
      CHECK(refused(call(a), code, word));
    };
    bad([](auto& a) { a.k = 0; }, EH_ERR_INVALID, "k:");
    bad([](auto& a) { a.k = 1025; }, EH_ERR_INVALID, "k:");
    bad([](auto& a) { a.k = 6; }, EH_ERR_SIZE, "teacher");
    bad([](auto& a) { a.temperature = 0; }, EH_ERR_INVALID, "temperature");
    bad([](auto& a) { a.temperature = 1e39; }, EH_ERR_INVALID, "temperature");
    bad([](auto& a) { a.temperature = 2e38; }, EH_ERR_INVALID, "temperature");       // 1 / it is denormal
    bad([](auto& a) { a.teacher.dtype = EH_I32; }, EH_ERR_INVALID, "teacher");
    bad([](auto& a) { a.ids.dtype = EH_F32; }, EH_ERR_INVALID, "ids");
    bad([](auto& a) { a.norm = eh_array{}; }, EH_ERR_INVALID, "norm");
    bad([](auto& a) { a.grad = a.logits; }, EH_ERR_INVALID, "overlap");
    eh_distill_loss_args a = ok;
    a.grad = eh_array{};
    CHECK(backward ? refused(call(a), EH_ERR_INVALID, "grad") : call(a) == EH_OK);
    a = ok;
    a.loss = eh_array{};
    CHECK(backward ? call(a) == EH_OK : refused(call(a), EH_ERR_INVALID, "loss"));
    a = ok;
    a.weight = eh_array{};
    CHECK(call(a) == EH_OK);
  }
}

static void recurrences(eh_device* d) {
  Pool p(d);
  eh_gated_scan_args ok{};
  ok.batch = 3, ok.time = 7, ok.width = 10, ok.log_gate = 1;
  ok.gate = p.array(3, 7, 10, EH_F16), ok.x = p.array(3, 7, 10, EH_F16), ok.out = p.array(3, 7, 10, EH_F16);
  ok.state = p.array(3, 1, 10, EH_F32), ok.final_state = p.array(3, 1, 10, EH_F32), ok.lengths = p.array(3, 1, 1, EH_I32);
  const int fills = g_fills;
  CHECK(eh_gated_scan(d, &ok, 0) == EH_OK);
  CHECK(g_fills == fills + 5);                   // with lengths the outputs keep what they hold: all but the final state
  auto bad = [&](auto change, int code, const char* word) {
    eh_gated_scan_args a = ok;
    change(a);
    CHECK(refused(eh_gated_scan(d, &a, 0), code, word));
  };
  bad([](auto& a) { a.batch = -1; }, EH_ERR_INVALID, "batch");
  bad([](auto& a) { a.time = -1; }, EH_ERR_INVALID, "time");
  bad([](auto& a) { a.width = 0; }, EH_ERR_INVALID, "width");
  bad([](auto& a) { a.batch = 1 << 22, a.width = 1 << 24; }, EH_ERR_INVALID, "batch, width");
  bad([](auto& a) { a.batch = 1 << 22, a.width = 2048, a.time = int64_t{1} << 31; }, EH_ERR_INVALID, "out of range together");
  bad([](auto& a) { a.x.dtype = EH_F32; }, EH_ERR_INVALID, "other arrays' type");
  bad([](auto& a) { a.out = a.x; }, EH_ERR_INVALID, "overlap");
  bad([](auto& a) { a.out.stride[1] = 9; }, EH_ERR_INVALID, "rows overlap");
  bad([](auto& a) { a.out.stride[0] = 69; }, EH_ERR_INVALID, "rows overlap");
  bad([](auto& a) { a.out.stride[0] = 0; }, EH_ERR_INVALID, "rows overlap");
  bad([](auto& a) { a.final_state = a.state; }, EH_ERR_INVALID, "overlap");
  bad([](auto& a) { a.lengths.dtype = EH_I64; }, EH_ERR_INVALID, "i32");
  bad([](auto& a) { a.x.stride[1] = 11; }, EH_ERR_SIZE, "size mismatch");
  eh_gated_scan_args a = ok;                     // steps outermost
  for (eh_array* x : {&a.gate, &a.x, &a.out}) x->stride[0] = 10, x->stride[1] = 30;
  CHECK(eh_gated_scan(d, &a, 0) == EH_OK);
  a = ok;                                        // one gate for all steps of all sequences
  a.gate.stride[0] = a.gate.stride[1] = 0;
  CHECK(eh_gated_scan(d, &a, 0) == EH_OK);
  a = ok;
  a.time = 0;
  CHECK(eh_gated_scan(d, &a, 0) == EH_OK);
  // gate, input and output as columns of one buffer
  a = ok;
  a.gate = p.array(3, 7, 30, EH_F16), a.x = a.gate, a.out = a.gate;
  a.x.offset = 20, a.out.offset = 40;
  CHECK(eh_gated_scan(d, &a, 0) == EH_OK);
  a.out.offset = 38;
  CHECK(eh_gated_scan(d, &a, 0) != EH_OK);
  eh_gated_scan_backward_args b{};
  b.batch = 3, b.time = 1100, b.width = 10;
  b.gate = p.array(3, 1100, 10, EH_F32), b.h = p.array(3, 1100, 10, EH_F32), b.grad_h = p.array(3, 1100, 10, EH_F32);
  b.grad_gate = p.array(3, 1100, 10, EH_F32), b.grad_x = p.array(3, 1100, 10, EH_F32);
  CHECK(eh_gated_scan_backward(d, &b, 0) == EH_OK);
  b.state = p.array(3, 1, 10, EH_F32), b.grad_state = p.array(3, 1, 10, EH_F32), b.grad_final = p.array(3, 1, 10, EH_F32);
  CHECK(eh_gated_scan_backward(d, &b, 0) == EH_OK);
  size_t n = 0;
  CHECK(eh_gated_scan_backward_workspace(d, &b, &n) == EH_OK && n > 0);
  b.workspace = p.array(1, 1, static_cast<int64_t>(n) / 4, EH_F32);
  CHECK(eh_gated_scan_backward(d, &b, 0) == EH_OK);
  b.grad_x = b.grad_gate;
  CHECK(refused(eh_gated_scan_backward(d, &b, 0), EH_ERR_INVALID, "overlap"));
}

// What the kernels take for granted of a plan, over many sizes.
static void plans() {
  uint64_t s = 88172645463325252ull;
  auto next = [&](int64_t lo, int64_t hi) {
    s ^= s << 13, s ^= s >> 7, s ^= s << 17;
    const double x = static_cast<double>(s >> 11) / 9007199254740992.0;
    return static_cast<int64_t>(static_cast<double>(lo) * std::pow(static_cast<double>(hi) / static_cast<double>(lo), x));
  };
  for (int i = 0; i < 200000; ++i) {
    const int dtype = i % 3, vec = 16 / static_cast<int>(elem_size(dtype));
    const int64_t rows = next(1, 1 << 24);
    const int vocab = static_cast<int>(next(1, 1 << 30));
    const bool top = i % 5 == 0;
    const RowSplit r = split_rows(rows, vocab, dtype, top, 256);
    bool ok = (r.threads == 64 || r.threads == 128 || r.threads == 256 || r.threads == 512 || r.threads == 1024) && r.segs >= 1;
    // the last segment is not empty, the others are whole, a launch's workgroups are countable
    ok = ok && static_cast<int64_t>(r.segs - 1) * r.seg < vocab && static_cast<int64_t>(r.segs) * r.seg >= vocab;
    ok = ok && (r.segs == 1 || (r.seg % vec == 0 && r.threads == 512)) && rows * r.segs < (int64_t{1} << 31);
    // a row held in registers fits them wherever it starts
    ok = ok && (!r.held || (!top && r.segs == 1 && held_form(r.threads, r.held) && static_cast<int64_t>(r.threads) * r.held * vec >= static_cast<int64_t>(vocab) + vec - 1));
    const RowHeld h = hold_rows(rows, vocab, dtype, 256);
    ok = ok && (h.vectors == 0 || static_cast<int64_t>(h.threads) * h.vectors >= vocab / vec);
    ok = ok && (h.vectors == 0 || (h.vectors == 4 && (h.threads == 64 || h.threads == 128 || h.threads == 256 || h.threads == 1024)) ||
                (h.vectors == 8 && h.threads == 256) || (h.vectors == 24 && h.threads == 1024) ||
                (h.vectors == 16 && (h.threads == 256 || h.threads == 512 || h.threads == 1024)));
    ScanArgs a{};
    a.compute_units = 256;
    a.dtype = dtype, a.batch = next(1, 1 << 16), a.time = next(1, int64_t{1} << 31), a.width = static_cast<int>(next(1, 1 << 18));
    a.gate.step = a.x.step = a.out.step = next(1, int64_t{1} << 40);
    const ScanPlan p = plan_scan(a);
    const int64_t wave = 64 / p.lanes * kScanSteps;
    ScanArgs close = a;                          // a workspace is asked for without the arrays' strides
    close.gate.step = close.x.step = close.out.step = a.width;
    ok = ok && scan_workspace(close) == scan_workspace(a) && scan_workspace(a) >= scan_board(a, p);
    ok = ok && (r.segs > 1 || r.held || top || r.threads >= 256);
    ok = ok && (p.lanes == 2 || p.lanes == 4 || p.lanes == 8) && (p.waves == 0 || p.waves == 1 || p.waves == 8 || (p.lanes == 8 && (p.waves == 2 || p.waves == 4 || (p.waves == 16 && p.pieces == 1)))) && (p.classes == 1 || p.classes == 8);
    ok = ok && (p.waves == 0 || (p.pieces * p.waves * wave >= a.time && (p.pieces - 1) * p.waves * wave < a.time));
    ok = ok && (p.pieces == 1 || p.waves == 8 || (p.waves == 0 && a.time <= 3 * kScanSteps)) && p.tiles * p.channels >= a.width && (p.tiles - 1) * p.channels < a.width;
    ok = ok && (p.waves == 0 || p.far || a.gate.step * static_cast<int64_t>(elem_size(dtype)) * (p.waves * wave + 1) < (int64_t{1} << 32)) && (!p.far || (p.lanes == 8 && (p.waves == 8 || p.waves == 0)));
    ok = ok && p.groups * p.per_group >= p.pieces && (p.waves != 8 || p.per_group * p.lanes == 128);
    ++g_checks;
    if (!ok) {
      ++g_failures;
      std::printf("plan: rows %lld vocab %d type %d, batch %lld time %lld width %d step %lld\n", static_cast<long long>(rows), vocab, dtype,
                  static_cast<long long>(a.batch), static_cast<long long>(a.time), a.width, static_cast<long long>(a.gate.step));
      if (g_failures > 20) return;
    }
  }
}

int main() {
  {
    eh_device d(0), other(0);
    scores(&d, &other);
    workspaces(&d);
    gradients(&d);
    distillation(&d);
    recurrences(&d);
    plans();
  }
  std::printf("%d checks, %d failed\n", g_checks, g_failures);
  return g_failures ? 1 : 0;
}
