// The language-model operators' kernels as the entry points (operators.cpp) see them: plain
// structures of device addresses and sizes, already checked, and one launch function each.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace eh {

enum ElemType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

inline size_t elem_size(int dtype) { return dtype == kF32 ? 4 : 2; }

constexpr int kMaxTop = 32;          // alternatives a row can report: one wave selects them among 64 groups
constexpr int kMaxTeacher = 1024;    // entries a teacher can give for a row: they are held in LDS

// Rows of logits: element (r, i) at z + (r * stride + i) elements.
struct LogitRows {
  const void* z;
  int64_t stride;
  int64_t rows;
  int vocab;
  int dtype;
  float scale;             // 1 / temperature
};

struct TokenIds {
  const void* ids;
  int wide;                // 64-bit integers
};

// How a pass over rows that reads each once goes to workgroups: a row to one of `threads` threads, or
// `segs` segments of `seg` elements with a second launch that joins them.
constexpr int kScoreHeld = 4;        // most items (16 bytes) of a thread in a row that is held in registers
constexpr bool held_form(int threads, int items) { return items == kScoreHeld || threads == 64 || (items == 3 && threads < 1024); }
struct RowSplit {
  int threads;
  int held;                // items a thread of a row held in registers (held_form), or 0
  int segs;
  int seg;
};
// A launch's threads are counted in 32 bits: most workgroups of 256 in one.
constexpr int64_t kLaunchBlocks = (int64_t{1} << 24) - 1;
RowSplit split_rows(int64_t rows, int vocab, int dtype, bool top, int compute_units);
// What a segment leaves for the join (its best keys, 8 bytes each, follow).
struct RowPartial {
  float largest, s, t, pad;
};
size_t split_workspace(const RowSplit& s, int64_t rows, int top);   // bytes; 0 for whole rows

// A row held in a workgroup's registers, `vectors` of 16 bytes a thread; 0 vectors: too long for that.
constexpr int kHeldInLds = 8;        // vectors of a thread in LDS besides 16 in registers, of the longest rows
struct RowHeld {
  int threads;
  int vectors;
};
RowHeld hold_rows(int64_t rows, int vocab, int dtype, int compute_units);

struct ScoreArgs {
  LogitRows in;
  TokenIds targets;
  int64_t ignore;
  float* logp;             // [rows]
  float* entropy;          // [rows] or null
  float* norm;             // [rows][2]: largest logit, log sum exp(scale (z - largest))
  float* top_logp;         // [rows][top]
  int* top_ids;
  int top;
  RowSplit split;
  void* workspace;
};
hipError_t launch_score(const ScoreArgs& a, hipStream_t stream);

struct ScoreGradArgs {
  LogitRows in;
  TokenIds targets;
  int64_t ignore;
  const float* norm;
  const float* entropy;        // null: no entropy gradient
  const float* grad_logp;      // null: none
  const float* grad_entropy;
  void* grad;
  int64_t grad_stride;
};
hipError_t launch_score_grad(const ScoreGradArgs& a, hipStream_t stream);

struct DistillArgs {
  LogitRows in;                // scale is 1 / temperature
  float temperature;
  const void* teacher;         // [rows][k], element type teacher_dtype
  int64_t teacher_stride;
  int teacher_dtype;
  TokenIds ids;                // [rows][k]
  int64_t ids_stride;
  int k;
  const float* weight;         // [rows] or null: what each row's gradient is multiplied by
  float* norm;                 // [rows][2]: written by the loss, read by the gradient alone
  float* loss;                 // [rows]
  void* grad;                  // null: no gradient
  int64_t grad_stride;
  RowSplit split;
  RowHeld held;
  void* workspace;
};
hipError_t launch_distill(const DistillArgs& a, hipStream_t stream);
hipError_t launch_distill_grad(const DistillArgs& a, hipStream_t stream);

// Element (b, t, d) at p + b * batch + t * step + d elements.
struct Sequences {
  void* p;
  int64_t batch, step;
};

struct ScanArgs {
  int64_t batch, time;
  int width;
  int dtype;
  int log_gate;                // gates are exp(gate)
  Sequences gate, x, out;      // gradients: gate, h (x) and grad_h (out) are read
  Sequences grad_gate, grad_x; // (gradients only)
  const float* state;          // [batch][width] or null (zeros)
  float* final_state;          // [batch][width] or null; gradients: the gradient of `state`
  const float* grad_final;     // gradients only, or null
  const int* lengths;          // [batch] or null
  int compute_units;
  void* workspace;
  unsigned int* lost;          // receives a 1 from a workgroup that has waited for another one in vain (host memory)
  bool lose_waits;             // (tests) leave a piece out, so that others wait for it in vain
};
// A workgroup of `waves` waves has `lanes` vectors of channels and a piece of waves * 64 / lanes * kScanSteps steps.
constexpr int kScanSteps = 8;        // of a thread
struct ScanPlan {
  int lanes;                         // side by side: 2, 4 or 8
  int waves;                         // 0: a thread has a whole sequence's steps of its channels
  bool far;                          // a piece's rows may lie further apart than 32-bit offsets reach
  int channels;                      // of a workgroup
  int64_t pieces, tiles;             // of a sequence, of a row
  int64_t per_group, groups;         // pieces whose maps are composed from one state
  int classes;                       // of columns, see the kernel
  bool wide;                         // gradients in 16 bits: all of a thread's loads at once, in twice the registers
};
ScanPlan plan_scan(const ScanArgs& a);
constexpr size_t kTicketBytes = 256;
size_t scan_board(const ScanArgs& a, const ScanPlan& p);      // bytes; 0 where a sequence is one piece
size_t scan_workspace(const ScanArgs& a);     // what sequences of these sizes may need, whatever their strides
hipError_t launch_scan(const ScanArgs& a, hipStream_t stream);
hipError_t launch_scan_grad(const ScanArgs& a, hipStream_t stream);

}  // namespace eh
