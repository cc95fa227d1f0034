// C entry points of the operators along time (see "operators along time over feature rows" in include/mfcc_amd.h).
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <numeric>
#include <type_traits>

#include "abi.h"
#include "sequence_kernels.h"

using mfcc::Batch;
using mfcc::fail;
using mfcc::Rows;

namespace {

constexpr int64_t kMaxColumns = 1 << 20;
constexpr int64_t kMaxSeqs = 1 << 24;
constexpr int64_t kMaxRows = 1 << 30;  // of one sequence: row numbers inside it are 32-bit
constexpr double kMaxValues = 1ll << 56;  // counts of values and bytes stay far inside 64 bits
constexpr int64_t kMaxStride = 1ll << 56;
constexpr int64_t kMaxThreads = UINT32_MAX;  // of one launch, in one direction of its grid: a launch counts threads in 32 bits

// The geometry of a call, checked once: 0 or a negative error code.
struct Shape {
  Batch b;
  int64_t longest, rows;  // most rows of one sequence; rows of all of them, padding included
};
int shape_of(const char* who, const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, int32_t reverse, Shape* out) {
  if (ncol < 1 || ncol > kMaxColumns) return fail(MFCC_ERR_INVALID, "%s: ncol=%d outside 1..%lld", who, ncol, (long long)kMaxColumns);
  if (time_steps < 0 || time_steps > INT32_MAX) return fail(MFCC_ERR_INVALID, "%s: time_steps=%lld outside 0..2^31-1", who, (long long)time_steps);
  if (layout) n_seq = layout->n_utts;
  if (n_seq < 0 || n_seq > kMaxSeqs) return fail(MFCC_ERR_INVALID, "%s: %lld sequences outside 0..2^24", who, (long long)n_seq);
  out->b = Batch{layout ? layout->d_frame_off : nullptr, layout ? layout->d_order : nullptr, n_seq, time_steps, ncol, reverse};
  out->longest = layout ? (time_steps ? std::min(layout->longest, time_steps) : layout->longest) : time_steps;
  out->rows = time_steps || !layout ? n_seq * time_steps : layout->total_frames;
  if (out->longest > kMaxRows) return fail(MFCC_ERR_UNSUPPORTED, "%s: a sequence of more than 2^30 rows", who);
  if ((double)out->rows * ncol > kMaxValues) return fail(MFCC_ERR_UNSUPPORTED, "%s: more than 2^56 values", who);
  return MFCC_OK;
}

int check_rows(const char* who, const char* name, const mfcc_rows* r, const Shape& s, bool output) {
  if (!r || (!r->data && s.rows > 0)) return fail(MFCC_ERR_INVALID, "%s: %s is null", who, name);
  if (r->row_stride < 0 || r->seq_stride < 0) return fail(MFCC_ERR_INVALID, "%s: negative stride of %s", who, name);
  if (r->row_stride > kMaxStride || r->seq_stride > kMaxStride) return fail(MFCC_ERR_INVALID, "%s: a stride of %s passes 2^56", who, name);
  if (output && s.rows > 1) {
    // rows of outputs do not overlap: one row after the other inside a sequence and sequence after sequence, or
    // time-major (all sequences' row t, then row t + 1)
    const int64_t nc = s.b.ncol, rs = r->row_stride, ss = r->seq_stride, n = s.b.n_seq, t = s.b.steps;
    const bool packed = t == 0;
    const bool ok = packed ? rs >= nc
                           : ((t == 1 || rs >= nc) && (n == 1 || ss >= (t - 1) * rs + nc)) || ((n == 1 || ss >= nc) && (t == 1 || rs >= (n - 1) * ss + nc));
    if (!ok) return fail(MFCC_ERR_INVALID, "%s: rows of %s overlap (row stride %lld, sequence stride %lld, %lld columns)", who, name,
                         (long long)rs, (long long)ss, (long long)nc);
  }
  return MFCC_OK;
}

// Where workgroups of one sequence are fewer than the compute units, sequences of many tiles are cut into pieces, and others spread over
// narrower column blocks.  Measured with 512 columns of bfloat16, forward (training step): one sequence of 512 rows (8 tiles)
// 11.1 (31.6) us whole, 12.8 (27.8) in pieces of 2 tiles; of 1024 rows 18.8 (56.6) and 13.8 (29.3), of 8192 rows 124 (396) and
// 18.3 (38.5).  32 sequences of up to 700 rows (11 tiles, 4 pieces would fill the card) 18.9 us whole, 28 in pieces.
// All sequences get the same number of pieces: one long one among many short ones gets few, and from 256 workgroups on none.
constexpr int64_t kFewBlocks = 256, kManyTiles = 10, kManyPieces = 5, kTargetBlocks = 512, kPieceTiles = 2;

// Workgroups of half the threads for the normalisation where there are many: half the slots to join a tile (10000 sequences of
// 299 rows of 39: 272 us with 512 threads, 228 with 256; 200 sequences of up to 1200 rows of 257, 1000 workgroups: 57 and 61).
constexpr int64_t kManyBlocks = 2048;
constexpr int kWideBlock = 40, kManySlots = 12;

// How workgroups divide sequences, columns and time.  It depends on the shape of the batch alone, so that the backward
// pass finds its checkpoints whatever the alignment of its arrays.
struct Grid {
  int v, tile_rows, threads;   // threads: of a workgroup, the waves that hold all its slots
  mfcc::Split w;
  dim3 blocks;
};
Grid grid_of(const Shape& s, int threads = mfcc::kSeqThreads) {
  Grid g;
  g.w.pieces = 1;
  g.w.near = 1;
  // column blocks of at most `wide` groups, equally wide; slots of time: as many as the threads give, at most 64 (each thread
  // composes the maps of all of them), and no more than the longest sequence fills; what is left over takes further sequences
  auto split = [&](int wide) {
    g.w.column_blocks = (g.w.groups + wide - 1) / wide;
    g.w.cb = (g.w.groups + g.w.column_blocks - 1) / g.w.column_blocks;
    const int slots = threads / g.w.cb;
    const int64_t need = std::max<int64_t>(1, (s.longest + mfcc::kSlotRows - 1) / mfcc::kSlotRows);
    g.w.per = (int32_t)std::min<int64_t>(std::min(slots, 64), need);
    g.w.seqs = need <= g.w.per ? slots / g.w.per : 1;
    g.tile_rows = g.w.per * mfcc::kSlotRows;
    g.w.blocks = (int32_t)blocks_for(s.b.n_seq, g.w.seqs);
    g.w.piece_tiles = (int32_t)std::max<int64_t>((s.longest + g.tile_rows - 1) / g.tile_rows, 1);
  };
  // values of a row that a thread takes at once: 2, but 1 for narrow rows with many slots of time, every one of which all threads
  // compose (10000 sequences of 300 rows of 40 bfloat16: 25 slots for 2 values 217 us forward and 547 back, 12 slots for 1 187 and 337)
  g.v = 2;
  g.w.groups = s.b.ncol / 2;
  if (s.b.ncol % 2 == 0) split(64);
  if (s.b.ncol % 2 || (g.w.cb < kWideBlock && g.w.per > kManySlots)) {
    g.v = 1;
    g.w.groups = s.b.ncol;
    split(64);   // at most a wave to a row
  }
  const int64_t blocks = (int64_t)g.w.blocks * g.w.column_blocks, tiles = g.w.piece_tiles;
  if (g.w.seqs == 1 && blocks > 0 && blocks < kFewBlocks) {
    const int64_t want = std::min(kTargetBlocks / blocks, tiles / kPieceTiles);   // not one more than the card takes at once
    if (tiles >= kManyTiles && want >= kManyPieces) {
      g.w.piece_tiles = (int32_t)((tiles + want - 1) / want);
      g.w.pieces = (int32_t)((tiles + g.w.piece_tiles - 1) / g.w.piece_tiles);
      g.w.blocks *= g.w.pieces;
    } else {
      split(32);   // twice the workgroups, of half the tiles (32 sequences of up to 700 rows: 23.6 -> 18.9 us)
    }
  }
  g.blocks = dim3((unsigned)((g.w.blocks + 7) / 8 * 8 * g.w.column_blocks));
  // 64 slots of fewer than 8 columns are not 8 waves (20000 sequences of 2000 floats: scan 218 us in one wave, 500 in eight)
  g.threads = std::min(threads, (g.w.seqs * g.w.per * g.w.cb + 63) / 64 * 64);
  return g;
}

// Floats of the checkpoints, bytes of the workspace.
int64_t checkpoints_of(const Shape& s, const Grid& g) {
  const int64_t k = g.tile_rows, t = s.b.steps;
  return (t || !s.b.off ? s.b.n_seq * ((t + k - 1) / k) : s.rows / k + s.b.n_seq) * s.b.ncol;
}
int64_t workspace_of(const Shape& s, const Grid& g) { return g.w.pieces > 1 ? s.b.n_seq * g.w.pieces * s.b.ncol * (int64_t)sizeof(mfcc::ScanMap) : 0; }

int check_grid(const char* who, const Shape& s, const Grid& g, const void* workspace) {
  if (((int64_t)g.w.blocks + 7) / 8 * 8 * g.w.column_blocks > kMaxThreads / g.threads)
    return fail(MFCC_ERR_UNSUPPORTED, "%s: %lld sequences of %d columns are more than one launch covers", who, (long long)s.b.n_seq, s.b.ncol);
  if (g.w.pieces > 1 && (!workspace || ((uintptr_t)workspace & 15)))
    return fail(MFCC_ERR_INVALID, "%s: this shape needs a 16-byte aligned workspace (mfcc_sequence_workspace)", who);
  return MFCC_OK;
}

bool aligned(const mfcc_rows* r, const Shape& s, int v, size_t size) {
  return !r || (((uintptr_t)r->data % (v * size)) == 0 && r->row_stride % v == 0 && (s.b.steps == 0 || r->seq_stride % v == 0));
}

// Offsets inside a tile (a piece) are 32-bit numbers of bytes where that is enough.
bool near(const mfcc_rows* r, const Grid& c, const Shape& s, size_t size) {
  const double rows = (double)c.tile_rows * (c.w.pieces > 1 ? c.w.piece_tiles : 1);
  return !r || (rows * (double)r->row_stride + s.b.ncol) * size < 4294967296.0;
}

// f(type's zero, number of values, aligned) for the row type, the values a thread takes and the alignment of the arrays
template <typename T, typename F>
void dispatch_pack(int v, bool al, F f) {
  if (v == 1) f((T)0.0f, std::integral_constant<int, 1>(), std::true_type());
  else if (al) f((T)0.0f, std::integral_constant<int, 2>(), std::true_type());
  else f((T)0.0f, std::integral_constant<int, 2>(), std::false_type());
}
template <typename F>
void dispatch(int32_t dtype, int v, bool al, F f) {
  if (dtype == MFCC_ROWS_F32) dispatch_pack<float>(v, al, f);
  else if (dtype == MFCC_ROWS_BF16) dispatch_pack<mfcc::bf16>(v, al, f);
  else dispatch_pack<mfcc::f16>(v, al, f);
}

// The array of rows for a kernel; null where the batch has no rows.
template <typename T>
Rows<T> rows_of(const mfcc_rows* r, const Shape& s) {
  return r && s.rows > 0 ? Rows<T>{(T*)r->data, r->seq_stride, r->row_stride} : Rows<T>{nullptr, 0, 0};
}

// The bytes that a call reads or writes through one argument: `seqs` blocks of `rows` rows of `width` bytes.
struct Bytes {
  const char* name;
  const char* p;
  int64_t width;
  int64_t row, seq;   // strides, 0 where there is but one
  int64_t rows, seqs;
};
Bytes bytes_of(const char* name, const mfcc_rows* r, const Shape& s, size_t size) {
  Bytes a{name, r && s.rows > 0 ? (const char*)r->data : nullptr, s.b.ncol * (int64_t)size, 0, 0, s.b.steps ? s.b.steps : s.rows, s.b.steps ? s.b.n_seq : 1};
  if (!a.p) return a;
  if (a.rows > 1) a.row = r->row_stride * (int64_t)size;
  if (a.seqs > 1) a.seq = r->seq_stride * (int64_t)size;
  return a;
}
Bytes bytes_of(const char* name, const void* p, int64_t bytes) { return Bytes{name, bytes > 0 ? (const char*)p : nullptr, bytes, 0, 0, 1, 1}; }

// No byte of a is one of b, as far as spans and strides tell: the whole spans, what lies between sequences, what lies between rows.
bool apart(const Bytes& a, const Bytes& b) {
  typedef __int128 wide;
  if (!a.p || !b.p) return true;
  const wide d = (wide)(intptr_t)b.p - (intptr_t)a.p;
  auto seq_span = [](const Bytes& x) { return (wide)(x.rows - 1) * x.row + x.width; };
  auto row_span = [](const Bytes& x) { return (wide)(x.seqs - 1) * x.seq + x.width; };
  if (d >= seq_span(a) + (wide)(a.seqs - 1) * a.seq || -d >= seq_span(b) + (wide)(b.seqs - 1) * b.seq) return true;
  auto between = [&](int64_t period, wide wa, wide wb) {   // both repeat with this period
    if (period <= 0) return false;
    const wide at = (d % period + period) % period;
    return at >= wa && period - at >= wb;
  };
  const int64_t seqs = std::gcd(a.seq, b.seq), rows = std::gcd(a.row, b.row);
  return between(seqs, seq_span(a), seq_span(b)) || between(rows, row_span(a), row_span(b)) || between(std::gcd(seqs, rows), a.width, b.width);
}
bool same(const Bytes& a, const Bytes& b) { return a.p == b.p && a.width == b.width && a.row == b.row && a.seq == b.seq; }

// Threads read and write in no order between workgroups: what a call writes lies apart from everything else, but for the arrays that it
// may work on in place.
int check_apart(const char* who, const Bytes& out, std::initializer_list<Bytes> others, bool in_place = false) {
  for (const Bytes& o : others)
    if (!apart(out, o) && !(in_place && same(out, o)))
      return fail(MFCC_ERR_INVALID, in_place ? "%s: %s overlaps %s without being the same rows" : "%s: %s overlaps %s", who, out.name, o.name);
  return MFCC_OK;
}

int bad_dtype(const char* who, int32_t dtype) { return fail(MFCC_ERR_INVALID, "%s: rows type %d", who, dtype); }

}  // namespace

extern "C" {

int64_t mfcc_gated_scan_checkpoints(const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, int32_t rows_dtype) {
  Shape s;
  if (const int rc = shape_of("mfcc_gated_scan_checkpoints", layout, n_seq, time_steps, ncol, 0, &s)) return rc;
  if (rows_dtype < 0 || rows_dtype > MFCC_ROWS_F16) return bad_dtype("mfcc_gated_scan_checkpoints", rows_dtype);
  return checkpoints_of(s, grid_of(s));
}

int64_t mfcc_sequence_workspace(const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, int32_t rows_dtype) {
  Shape s;
  if (const int rc = shape_of("mfcc_sequence_workspace", layout, n_seq, time_steps, ncol, 0, &s)) return rc;
  if (rows_dtype < 0 || rows_dtype > MFCC_ROWS_F16) return bad_dtype("mfcc_sequence_workspace", rows_dtype);
  return workspace_of(s, grid_of(s));
}

int mfcc_gated_scan(const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, int32_t rows_dtype, int32_t form,
                    int32_t reverse, const mfcc_rows* x, const mfcc_rows* gate, const float* h0, const mfcc_rows* y, float* last,
                    float* checkpoints, void* workspace, void* stream) {
  static const char who[] = "mfcc_gated_scan";
  Shape s;
  if (const int rc = shape_of(who, layout, n_seq, time_steps, ncol, reverse ? 1 : 0, &s)) return rc;
  if (form != MFCC_SCAN_DECAY && form != MFCC_SCAN_SIGMOID) return fail(MFCC_ERR_INVALID, "%s: form=%d", who, form);
  if (const int rc = check_rows(who, "x", x, s, false)) return rc;
  if (const int rc = check_rows(who, "gate", gate, s, false)) return rc;
  if (const int rc = check_rows(who, "y", y, s, true)) return rc;
  if (rows_dtype < 0 || rows_dtype > MFCC_ROWS_F16) return bad_dtype(who, rows_dtype);
  if (s.b.n_seq == 0) return MFCC_OK;
  Grid c = grid_of(s);
  if (const int rc = check_grid(who, s, c, workspace)) return rc;
  const mfcc::ScanPtrs q{h0, nullptr, last, checkpoints, nullptr, (mfcc::ScanMap*)workspace};
  const size_t size = rows_dtype == MFCC_ROWS_F32 ? 4 : 2;
  {
    const int64_t ends = s.b.n_seq * ncol * (int64_t)sizeof(float);
    const Bytes bx = bytes_of("x", x, s, size), bg = bytes_of("gate", gate, s, size), by = bytes_of("y", y, s, size), bh = bytes_of("h0", h0, ends),
                bl = bytes_of("last", last, ends), bc = bytes_of("checkpoints", checkpoints, checkpoints_of(s, c) * (int64_t)sizeof(float)),
                bw = bytes_of("workspace", workspace, workspace_of(s, c));
    if (const int rc = check_apart(who, by, {bx, bg}, true)) return rc;
    if (const int rc = check_apart(who, bl, {bx, bg, by, bh})) return rc;
    if (const int rc = check_apart(who, by, {bh})) return rc;
    if (const int rc = check_apart(who, bc, {bx, bg, by, bh, bl})) return rc;
    if (const int rc = check_apart(who, bw, {bx, bg, by, bh, bl, bc})) return rc;
  }
  const bool al = aligned(x, s, c.v, size) && aligned(gate, s, c.v, size) && aligned(y, s, c.v, size);
  c.w.near = near(x, c, s, size) && near(gate, c, s, size) && near(y, c, s, size);
  dispatch(rows_dtype, c.v, al, [&](auto zero, auto v, auto al) {
    using T = decltype(zero);
    if (c.w.pieces > 1) {
      auto k = form == MFCC_SCAN_SIGMOID ? mfcc::gated_scan_pieces_kernel<T, v(), al(), true, false>
                                         : mfcc::gated_scan_pieces_kernel<T, v(), al(), false, false>;
      hipLaunchKernelGGL(k, c.blocks, dim3(c.threads), 0, (hipStream_t)stream, s.b, c.w, rows_of<const T>(x, s), rows_of<const T>(gate, s), q);
    }
    auto k = form == MFCC_SCAN_SIGMOID ? mfcc::gated_scan_kernel<T, v(), al(), true> : mfcc::gated_scan_kernel<T, v(), al(), false>;
    hipLaunchKernelGGL(k, c.blocks, dim3(c.threads), 0, (hipStream_t)stream, s.b, c.w, rows_of<const T>(x, s), rows_of<const T>(gate, s),
                       rows_of<T>(y, s), q);
  });
  HIP_TRY(hipGetLastError());
  return MFCC_OK;
}

int mfcc_gated_scan_backward(const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, int32_t rows_dtype, int32_t form,
                             int32_t reverse, const mfcc_rows* x, const mfcc_rows* gate, const float* checkpoints,
                             const mfcc_rows* grad_y, const float* grad_last, const mfcc_rows* grad_x, const mfcc_rows* grad_gate,
                             float* grad_h0, void* workspace, void* stream) {
  static const char who[] = "mfcc_gated_scan_backward";
  Shape s;
  if (const int rc = shape_of(who, layout, n_seq, time_steps, ncol, reverse ? 1 : 0, &s)) return rc;
  if (form != MFCC_SCAN_DECAY && form != MFCC_SCAN_SIGMOID) return fail(MFCC_ERR_INVALID, "%s: form=%d", who, form);
  if (const int rc = check_rows(who, "x", x, s, false)) return rc;
  if (const int rc = check_rows(who, "gate", gate, s, false)) return rc;
  if (grad_y)
    if (const int rc = check_rows(who, "grad_y", grad_y, s, false)) return rc;
  if (const int rc = check_rows(who, "grad_x", grad_x, s, true)) return rc;
  if (const int rc = check_rows(who, "grad_gate", grad_gate, s, true)) return rc;
  if (!checkpoints && s.rows > 0) return fail(MFCC_ERR_INVALID, "%s: checkpoints is null", who);
  if (rows_dtype < 0 || rows_dtype > MFCC_ROWS_F16) return bad_dtype(who, rows_dtype);
  if (s.b.n_seq == 0) return MFCC_OK;
  Grid c = grid_of(s);
  if (const int rc = check_grid(who, s, c, workspace)) return rc;
  const mfcc::ScanPtrs q{nullptr, grad_last, nullptr, const_cast<float*>(checkpoints), grad_h0, (mfcc::ScanMap*)workspace};
  const size_t size = rows_dtype == MFCC_ROWS_F32 ? 4 : 2;
  {
    const int64_t ends = s.b.n_seq * ncol * (int64_t)sizeof(float);
    const Bytes bx = bytes_of("x", x, s, size), bg = bytes_of("gate", gate, s, size), bd = bytes_of("grad_y", grad_y, s, size),
                bl = bytes_of("grad_last", grad_last, ends), bc = bytes_of("checkpoints", checkpoints, checkpoints_of(s, c) * (int64_t)sizeof(float)),
                gx = bytes_of("grad_x", grad_x, s, size), gg = bytes_of("grad_gate", grad_gate, s, size), gh = bytes_of("grad_h0", grad_h0, ends),
                bw = bytes_of("workspace", workspace, workspace_of(s, c));
    if (const int rc = check_apart(who, gx, {bx, bg, bd, bl, bc})) return rc;
    if (const int rc = check_apart(who, gg, {bx, bg, bd, bl, bc, gx})) return rc;
    if (const int rc = check_apart(who, gh, {bx, bg, bd, bl, bc, gx, gg})) return rc;
    if (const int rc = check_apart(who, bw, {bx, bg, bd, bl, bc, gx, gg, gh})) return rc;
  }
  const bool al = aligned(x, s, c.v, size) && aligned(gate, s, c.v, size) && aligned(grad_y, s, c.v, size) && aligned(grad_x, s, c.v, size) &&
            aligned(grad_gate, s, c.v, size);
  c.w.near = near(x, c, s, size) && near(gate, c, s, size) && near(grad_y, c, s, size) && near(grad_x, c, s, size) && near(grad_gate, c, s, size);
  dispatch(rows_dtype, c.v, al, [&](auto zero, auto v, auto al) {
    using T = decltype(zero);
    if (c.w.pieces > 1) {
      auto k = form == MFCC_SCAN_SIGMOID ? mfcc::gated_scan_pieces_kernel<T, v(), al(), true, true>
                                         : mfcc::gated_scan_pieces_kernel<T, v(), al(), false, true>;
      hipLaunchKernelGGL(k, c.blocks, dim3(c.threads), 0, (hipStream_t)stream, s.b, c.w, rows_of<const T>(grad_y, s),
                         rows_of<const T>(gate, s), q);
    }
    auto k = form == MFCC_SCAN_SIGMOID ? mfcc::gated_scan_backward_kernel<T, v(), al(), true> : mfcc::gated_scan_backward_kernel<T, v(), al(), false>;
    hipLaunchKernelGGL(k, c.blocks, dim3(c.threads), 0, (hipStream_t)stream, s.b, c.w, rows_of<const T>(x, s), rows_of<const T>(gate, s),
                       rows_of<const T>(grad_y, s), rows_of<T>(grad_x, s), rows_of<T>(grad_gate, s), q);
  });
  HIP_TRY(hipGetLastError());
  return MFCC_OK;
}

int mfcc_gated_scan_step(int64_t n_seq, int32_t ncol, int32_t rows_dtype, int32_t form, const void* x, int64_t x_ld, const void* gate,
                         int64_t gate_ld, const float* state_in, float* state_out, void* y, int64_t y_ld, void* stream) {
  static const char who[] = "mfcc_gated_scan_step";
  if (ncol < 1 || ncol > kMaxColumns || n_seq < 0 || n_seq > INT32_MAX || x_ld < 0 || gate_ld < 0 ||
      std::max({x_ld, gate_ld, y_ld}) > kMaxStride)
    return fail(MFCC_ERR_INVALID, "%s: bad shape", who);
  if (n_seq > 1 && y_ld < ncol) return fail(MFCC_ERR_INVALID, "%s: rows of y overlap", who);
  if (form != MFCC_SCAN_DECAY && form != MFCC_SCAN_SIGMOID) return fail(MFCC_ERR_INVALID, "%s: form=%d", who, form);
  if (n_seq == 0) return MFCC_OK;
  if (n_seq * ncol > kMaxThreads - 255) return fail(MFCC_ERR_UNSUPPORTED, "%s: too many values per call", who);
  if (!x || !gate || !state_in || !state_out || !y) return fail(MFCC_ERR_INVALID, "%s: null pointer", who);
  if (rows_dtype < 0 || rows_dtype > MFCC_ROWS_F16) return bad_dtype(who, rows_dtype);
  {
    // a thread reads its element everywhere before it writes it: any of the arrays may be one and the same
    const int64_t size = rows_dtype == MFCC_ROWS_F32 ? 4 : 2;
    auto rows = [&](const char* name, const void* p, int64_t e, int64_t ld) { return Bytes{name, (const char*)p, ncol * e, n_seq > 1 ? ld * e : 0, 0, n_seq, 1}; };
    const Bytes bx = rows("x", x, size, x_ld), bg = rows("gate", gate, size, gate_ld), by = rows("y", y, size, y_ld),
                bi = rows("state_in", state_in, 4, ncol), bo = rows("state_out", state_out, 4, ncol);
    if (const int rc = check_apart(who, by, {bx, bg, bi, bo}, true)) return rc;
    if (const int rc = check_apart(who, bo, {bx, bg, bi}, true)) return rc;
  }
  auto go = [&](auto zero) {
    using T = decltype(zero);
    auto k = form == MFCC_SCAN_SIGMOID ? mfcc::gated_scan_step_kernel<T, true> : mfcc::gated_scan_step_kernel<T, false>;
    hipLaunchKernelGGL(k, dim3(blocks_for(n_seq * ncol, 256)), dim3(256), 0, (hipStream_t)stream, n_seq, ncol, (const T*)x, x_ld,
                       (const T*)gate, gate_ld, state_in, state_out, (T*)y, y_ld);
  };
  if (rows_dtype == MFCC_ROWS_F32) go(0.0f);
  else if (rows_dtype == MFCC_ROWS_BF16) go((mfcc::bf16)0.0f);
  else go((mfcc::f16)0.0f);
  HIP_TRY(hipGetLastError());
  return MFCC_OK;
}

int mfcc_running_norm(const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, double decay, double eps,
                      int32_t center_only, const mfcc_rows* x, const float* state_in, const mfcc_rows* y, int32_t y_dtype,
                      float* state_out, void* workspace, void* stream) {
  static const char who[] = "mfcc_running_norm";
  Shape s;
  if (const int rc = shape_of(who, layout, n_seq, time_steps, ncol, 0, &s)) return rc;
  if (!(decay > 0.0 && decay <= 1.0)) return fail(MFCC_ERR_INVALID, "%s: decay=%g outside (0, 1]", who, decay);
  if (!(eps >= 0.0 && eps <= 1e30)) return fail(MFCC_ERR_INVALID, "%s: eps=%g", who, eps);
  if (const int rc = check_rows(who, "x", x, s, false)) return rc;
  if (const int rc = check_rows(who, "y", y, s, true)) return rc;
  if (y_dtype < 0 || y_dtype > MFCC_ROWS_F16) return bad_dtype(who, y_dtype);
  if (s.b.n_seq == 0) return MFCC_OK;
  Grid c = grid_of(s);
  if (const int rc = check_grid(who, s, c, workspace)) return rc;
  if (c.w.pieces == 1 && (int64_t)c.w.blocks * c.w.column_blocks >= kManyBlocks) {
    c = grid_of(s, mfcc::kSeqThreads / 2);
    if (const int rc = check_grid(who, s, c, workspace)) return rc;
  }
  const size_t size = y_dtype == MFCC_ROWS_F32 ? 4 : 2;
  {
    const int64_t ends = s.b.n_seq * (1 + 2 * (int64_t)ncol) * (int64_t)sizeof(float);
    const Bytes bx = bytes_of("x", x, s, 4), by = bytes_of("y", y, s, size), bi = bytes_of("state_in", state_in, ends),
                bo = bytes_of("state_out", state_out, ends), bw = bytes_of("workspace", workspace, workspace_of(s, c));
    if (const int rc = check_apart(who, by, {bx}, true)) return rc;
    if (const int rc = check_apart(who, by, {bi})) return rc;
    if (const int rc = check_apart(who, bo, {bx, by, bi})) return rc;
    if (const int rc = check_apart(who, bw, {bx, by, bi, bo})) return rc;
  }
  const bool al = aligned(x, s, c.v, 4) && aligned(y, s, c.v, size);
  c.w.near = near(x, c, s, 4) && near(y, c, s, size);
  mfcc::NormArgs a;
  a.decay = decay;
  a.log_decay = std::log1p(decay - 1.0);
  auto weights = [&](double k, double* decayed, double* grown) {
    const double em = std::expm1(k * a.log_decay);
    *decayed = 1.0 + em;
    *grown = decay == 1.0 ? k : em / (decay - 1.0);
  };
  weights(mfcc::kSlotRows, &a.slot_decay, &a.slot_grown);
  weights(c.tile_rows, &a.tile_decay, &a.tile_grown);
  weights((double)c.w.piece_tiles * mfcc::kSlotRows, &a.run_decay, &a.run_grown);
  weights((double)c.w.piece_tiles * c.tile_rows, &a.piece_decay, &a.piece_grown);
  for (int r = 0; r < mfcc::kSlotRows; ++r) {
    double l, g;
    weights(r + 1, &l, &g);
    a.decayed[r] = (float)l;
    a.grown[r] = (float)g;
    a.inv_grown[r] = (float)(1.0 / g);
  }
  a.eps = (float)eps;
  a.center_only = center_only ? 1 : 0;
  a.state_in = state_in;
  a.state_out = state_out;
  a.runs = (float2*)workspace;
  dispatch(y_dtype, c.v, al, [&](auto zero, auto v, auto al) {
    using T = decltype(zero);
    if (c.w.pieces > 1)
      hipLaunchKernelGGL((mfcc::running_norm_pieces_kernel<v(), al()>), c.blocks, dim3(c.threads), 0, (hipStream_t)stream, s.b, c.w, rows_of<const float>(x, s), a);
    const int slots = c.w.seqs * c.w.per;
    const size_t shared = 2 * slots * ((1 + mfcc::kSlotRows / 4) * sizeof(float4) + v() * c.w.cb * sizeof(float2));
    auto k = a.eps < 0x1p-126f && !center_only ? mfcc::running_norm_kernel<T, v(), al(), true> : mfcc::running_norm_kernel<T, v(), al(), false>;
    hipLaunchKernelGGL(k, c.blocks, dim3(c.threads), shared, (hipStream_t)stream, s.b, c.w, rows_of<const float>(x, s), rows_of<T>(y, s), a);
  });
  HIP_TRY(hipGetLastError());
  return MFCC_OK;
}

int mfcc_feature_dropout(const mfcc_layout* layout, int64_t n_seq, int64_t time_steps, int32_t ncol, int32_t rows_dtype, int32_t per,
                         int32_t threshold, uint64_t seed, uint64_t step, const int64_t* step_device, const mfcc_rows* x,
                         const mfcc_rows* y, void* stream) {
  static const char who[] = "mfcc_feature_dropout";
  Shape s;
  if (const int rc = shape_of(who, layout, n_seq, time_steps, ncol, 0, &s)) return rc;
  if (per < MFCC_DROP_ELEMENT || per > MFCC_DROP_SEQUENCE) return fail(MFCC_ERR_INVALID, "%s: per=%d", who, per);
  if (threshold < 0 || threshold > 65536) return fail(MFCC_ERR_INVALID, "%s: threshold=%d outside 0..65536", who, threshold);
  if (const int rc = check_rows(who, "x", x, s, false)) return rc;
  if (const int rc = check_rows(who, "y", y, s, true)) return rc;
  if (s.rows == 0) return MFCC_OK;
  if (rows_dtype < 0 || rows_dtype > MFCC_ROWS_F16) return bad_dtype(who, rows_dtype);
  const mfcc::Dropout d{seed, step, step_device, (uint32_t)threshold, threshold < 65536 ? 65536.0f / (float)(65536 - threshold) : 0.0f};
  const size_t size = rows_dtype == MFCC_ROWS_F32 ? 4 : 2;
  const int64_t most = (int64_t)INT32_MAX * 8;
  {
    const Bytes by = bytes_of("y", y, s, size);
    if (const int rc = check_apart(who, by, {bytes_of("x", x, s, size)}, true)) return rc;
    if (const int rc = check_apart(who, by, {bytes_of("step_device", step_device, sizeof(int64_t))})) return rc;
  }
  hipStream_t st = (hipStream_t)stream;
  // a batch without padding between its rows is one run of rows
  auto flat = [&](const mfcc_rows* r) {
    return r->row_stride == ncol && (s.b.steps == 0 || s.b.n_seq == 1 || r->seq_stride == s.b.steps * ncol) && (uintptr_t)r->data % 16 == 0;
  };
  if (per == MFCC_DROP_ELEMENT) {
    const int64_t blocks = (s.rows * ncol + 8 * 256 - 1) / (8 * 256);
    if (blocks > kMaxThreads / 256) return fail(MFCC_ERR_UNSUPPORTED, "%s: too many rows per call", who);
    const bool fl = flat(x) && flat(y);
    dispatch(rows_dtype, 1, true, [&](auto zero, auto, auto) {
      using T = decltype(zero);
      auto k = fl ? mfcc::dropout_element_kernel<T, true> : mfcc::dropout_element_kernel<T, false>;
      hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, s.b, s.rows, d, rows_of<const T>(x, s), rows_of<T>(y, s));
    });
  } else {
    const int v = ncol % 2 == 0 && aligned(x, s, 2, size) && aligned(y, s, 2, size) ? 2 : 1;
    mfcc::Split w{};
    w.groups = ncol / v;
    w.column_blocks = (w.groups + 255) / 256;
    w.cb = (w.groups + w.column_blocks - 1) / w.column_blocks;
    w.per = 256 / w.cb;
    if (s.rows > most || w.column_blocks > 65535) return fail(MFCC_ERR_UNSUPPORTED, "%s: too many rows or columns per call", who);
    // groups of 8 rows to a thread: per frame 1; per sequence as many as leave the card 2048 workgroups, but 1 where the 8 rows of a few
    // columns are far from the next thread's (10000 x 300 rows of 39 bfloat16: per frame 1 group 4.0 TB/s, 8 groups 3.5; per sequence
    // 1.6 and 3.1; 20000 x 500 rows of 4 floats per sequence 3.0 and 2.7, of 8 floats 3.8 and 3.5, 10000 x 300 of 13 2.5 and 3.0)
    const int64_t groups = (s.rows + 7) / 8;
    const bool frame = per == MFCC_DROP_FRAME;
    int runs = frame || w.cb < 8 ? 1 : 8;
    while (runs > 1 && groups / (w.per * runs) * w.column_blocks < 2048) runs /= 2;
    if ((groups + w.per * runs - 1) / (w.per * runs) > kMaxThreads / 256) return fail(MFCC_ERR_UNSUPPORTED, "%s: too many rows per call", who);
    const dim3 grid(blocks_for(groups, w.per * runs), (unsigned)w.column_blocks);
    auto linear = [&](const mfcc_rows* r) { return s.b.steps == 0 || s.b.n_seq == 1 || r->seq_stride == s.b.steps * r->row_stride; };
    const bool lin = linear(x) && linear(y);
    dispatch(rows_dtype, v, true, [&](auto zero, auto vv, auto) {
      using T = decltype(zero);
      auto k = frame ? (lin ? mfcc::dropout_rows_kernel<T, vv(), true, true> : mfcc::dropout_rows_kernel<T, vv(), true, false>)
                     : (lin ? mfcc::dropout_rows_kernel<T, vv(), false, true> : mfcc::dropout_rows_kernel<T, vv(), false, false>);
      hipLaunchKernelGGL(k, grid, dim3(256), 0, st, s.b, w, runs, s.rows, d, rows_of<const T>(x, s), rows_of<T>(y, s));
    });
  }
  HIP_TRY(hipGetLastError());
  return MFCC_OK;
}

}  // extern "C"
