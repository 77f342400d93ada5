// How the language-model operators' launches are cut: rules on sizes and types alone.
#include <algorithm>

#include "operators.hpp"

namespace eh {

// Measured on 256 compute units, us a call:
//   few rows                     many rows, short                       many rows, long
//   8 x 32000 bf16               16384 x 1000 bf16                      4096 x 50264 bf16, 20 alternatives
//   256 threads 11.2, 1024 10.6   64 threads 10.3, 128 13.0, 256 20      256 threads 105, 512 96, 1024 175
// and 1021 x 50257 f16 with 5: 256 threads 27, 512 34 (its workgroups are all on the device at once, more
// threads only lengthen the selection).  Segments only pay where a row is long and there are few:
// 1 x 150000 f32 11.7 against 15.6 with one workgroup of 1024, 64 x 150000 bf16 16.6 against 17.8.
// Without alternatives a row goes to the registers of the smallest workgroup that holds it, us against the kernel
// that streams, 16384 rows: x 500 bf16 8.1 : 10.2, 2000 14 : 22, 6000 33 : 37, 8000 39 : 50, 12000 78 : 77, 16000
// 93 : 101, f32 x 4000 37 : 43; with 1024 threads only few rows (8192 x 32000 bf16 107 : 97, 8 x 32000 7.3 : 7.5).
RowSplit split_rows(int64_t rows, int vocab, int dtype, bool top, int compute_units) {
  const int vec = 16 / static_cast<int>(elem_size(dtype));
  const int64_t items = (vocab + vec - 1) / vec, held = items + 1;       // one more where a row starts between two
  if (items > 32768 && rows * 4 <= compute_units) {
    // 32 KB a segment at least, four vectors for each of 512 threads
    const int64_t want = (2 * static_cast<int64_t>(compute_units) + rows - 1) / rows;
    const int64_t segs = std::min<int64_t>(want, items / 2048);
    const int64_t seg = (items + segs - 1) / segs * vec;
    return {512, 0, static_cast<int>((vocab + seg - 1) / seg), static_cast<int>(seg)};
  }
  if (!top) {
    for (int threads = 64; threads <= (rows <= compute_units ? 1024 : 512); threads *= 2)
      for (int n = 1; n <= kScoreHeld; ++n)
        if (held_form(threads, n) && held <= n * threads) return {threads, n, 1, vocab};
  }
  if (rows <= compute_units) return {items <= 256 ? 64 : items <= 512 ? 128 : items <= 1024 ? 256 : items <= 2048 ? 512 : 1024, 0, 1, vocab};
  if (items <= 512) return {64, 0, 1, vocab};
  if (items <= 2048 && top) return {128, 0, 1, vocab};
  return {items > 4096 && rows >= 8 * static_cast<int64_t>(compute_units) ? 512 : 256, 0, 1, vocab};
}

size_t split_workspace(const RowSplit& s, int64_t rows, int top) {
  if (s.segs == 1) return 0;
  return static_cast<size_t>(rows) * static_cast<size_t>(s.segs) * (sizeof(RowPartial) + 8 * static_cast<size_t>(top));
}

// The smallest workgroup that holds a row, with few rows the largest (us a call):
//   16384 x 1000 bf16     64 x 4 20.9, 256 x 4 49         4096 x 64000 bf16   512 x 16 204, 1024 x 16 245
//   4096 x 32000 bf16    256 x 16 108, 1024 x 16 156      256 x 32000 bf16    1024 x 4 11.9, 256 x 16 13.8
//   16384 x 4000 bf16    128 x 4 49, 256 x 4 59           8192 x 12000 bf16   256 x 8 78, 256 x 16 88 (8192 x 8000 f32 103, 97)
//   8192 x 190000 bf16   1024 x (16 + 8 in LDS) 1278, in two readings 1546, as rows that are longer still are taken
RowHeld hold_rows(int64_t rows, int vocab, int dtype, int compute_units) {
  const int64_t vectors = vocab / (16 / static_cast<int64_t>(elem_size(dtype)));
  if (vectors <= 256) return {64, 4};
  if (rows <= 2 * static_cast<int64_t>(compute_units) && vectors <= 4096) return {1024, 4};
  if (vectors <= 512) return {128, 4};
  if (vectors <= 1024) return {256, 4};
  if (vectors <= 2048 && dtype != kF32) return {256, 8};
  if (vectors <= 4096) return {256, 16};
  if (vectors <= 8192) return {512, 16};
  if (vectors <= 16384) return {1024, 16};
  if (vectors <= 1024 * (16 + kHeldInLds)) return {1024, 16 + kHeldInLds};
  return {1024, 0};
}

// Whether every row starts at a cache line.
static bool on_lines(const Sequences& s, const ScanArgs& a) {
  const int64_t size = static_cast<int64_t>(elem_size(a.dtype));
  return reinterpret_cast<uintptr_t>(s.p) % 128 == 0 && (a.time <= 1 || s.step * size % 128 == 0) && (a.batch <= 1 || s.batch * size % 128 == 0);
}

// Sequences of a few steps by a thread each, where that fills the device (1024 x 9 x 2048 bf16 20 us against 69
// with a piece's 64 steps for each, 64 x 16 x 2048 8 us against 8.5, from 32 steps on no difference).
// One piece of 16 waves instead of two of 8 with a board: 16 x 700 x 2048 bf16 32 us against 36, 64 x 520 x 1024 57
// against 64, but many of all 1024 steps 32 x 1000 x 2048 96 against 88 (one workgroup on a compute unit).
// Wide: one workgroup on a compute unit instead of two, us a gradient with and without, by workgroups of a compute unit:
//   one    4 x 1999 x 717 f16 20.2 : 21.5, 2 x 4096 x 1024 bf16 23.1 : 24.1
//   two    4 x 4096 x 1024 bf16 49.5 : 49.4, 32 x 512 x 704 f16 34 : 31     three  24 x 512 x 2048 f16 64 : 59
//   four   32 x 512 x 2048 f16 81 : 80          five  40 x 512 x 2048 f16 98 : 97
//   six    48 x 512 x 2048 f16 114.6 : 115.3    seven 7 x 4096 x 2048 bf16 128.5 : 129.2
//   eight  8 x 4096 x 2048 bf16 144 : 147, 64 x 512 x 2048 f16 148 : 151     ten    20 x 4096 x 1024 bf16 174 : 179
//   more   16 x 4096 x 2048 bf16 261 : 273, 52 x 2048 x 717 f16 215 : 224, 64 x 4096 x 2048 bf16 960 : 1014
// From two to five it loses or is even, at six and seven the sides differ by less than one in a hundred.
// (in f32, which needs fewer registers, 161 : 156 and 497 : 502)
ScanPlan plan_scan(const ScanArgs& a) {
  ScanPlan p{};
  int64_t step = 0;
  for (int64_t s : {a.gate.step, a.x.step, a.out.step, a.grad_gate.step, a.grad_x.step}) step = std::max(step, s);
  const int64_t vectors = (a.width * static_cast<int64_t>(elem_size(a.dtype)) + 15) / 16;
  p.lanes = vectors <= 2 ? 2 : vectors <= 4 ? 4 : 8;
  const int64_t wave = 64 / p.lanes * kScanSteps;
  int64_t piece = wave;
  if (a.time > kScanSteps && (a.time > 3 * kScanSteps || a.batch * vectors < (1 << 16))) {
    const int64_t tiles = (vectors + p.lanes - 1) / p.lanes;
    if (a.time <= wave) p.waves = 1;
    else if (p.lanes < 8) p.waves = 8;
    else if (a.time <= 2 * wave) p.waves = 2;
    else if (a.time <= 4 * wave) p.waves = 4;
    else if (a.time <= 8 * wave) p.waves = 8;
    else p.waves = a.time <= 10 * wave || (a.time <= 16 * wave && a.batch * tiles <= 2 * static_cast<int64_t>(a.compute_units)) ? 16 : 8;
    piece = p.waves * wave;
    // (the rows of a piece and the one before them)
    p.far = step * static_cast<int64_t>(elem_size(a.dtype)) * (piece + 1) >= (int64_t{1} << 32);
    if (p.far) p.lanes = 8, p.waves = 8, piece = 8 * 64;
  }
  p.channels = p.lanes * (16 / static_cast<int>(elem_size(a.dtype)));
  p.tiles = (a.width + p.channels - 1) / p.channels;
  p.pieces = std::max<int64_t>((a.time + piece - 1) / piece, 1);
  p.per_group = p.waves == 8 ? 128 / p.lanes : 1;                       // 512 threads read one word each in f32, two in 16 bits
  p.groups = (p.pieces + p.per_group - 1) / p.per_group;
  bool lines = true;
  for (const Sequences* s : {&a.gate, &a.x, &a.out, &a.grad_gate, &a.grad_x})
    if (s->p) lines = lines && on_lines(*s, a);
  p.classes = lines ? 1 : 8;
  const int64_t blocks = a.batch * p.tiles * p.pieces;
  p.wide = blocks <= a.compute_units || blocks >= 8 * static_cast<int64_t>(a.compute_units);
  return p;
}

size_t scan_board(const ScanArgs& a, const ScanPlan& p) {
  if (p.pieces == 1) return 0;
  return kTicketBytes + static_cast<size_t>(a.batch * p.tiles) * static_cast<size_t>(p.channels) *
                            (8 * static_cast<size_t>(p.pieces) + 4 * static_cast<size_t>(p.groups));
}

size_t scan_workspace(const ScanArgs& a) {
  ScanArgs apart = a;
  apart.gate.step = int64_t{1} << 40;
  return std::max(scan_board(a, plan_scan(a)), scan_board(apart, plan_scan(apart)));
}

}  // namespace eh
