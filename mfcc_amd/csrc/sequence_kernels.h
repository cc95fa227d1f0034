// Operators along time over feature rows: the gated recurrence with its gradient, the running
// mean / variance normalisation and the dropout whose mask is never stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace mfcc {

typedef __bf16 bf16;
typedef _Float16 f16;

// One array of rows: element (sequence u, row t, column c), see mfcc_rows.
template <typename T>
struct Rows {
  T* p;
  int64_t ss, rs;
};

struct Batch {
  const int64_t* off;  // packed rows / lengths; nullptr: steps rows each
  const int64_t* order;  // the sequences by falling length, so that the longest start first; nullptr: as they come
  int64_t n_seq;
  int64_t steps;       // 0 = packed
  int32_t ncol;
  int32_t reverse;
};

// Rows of sequence u, and the row of the array that its first one is.
struct Span {
  int64_t first, n;
};
__device__ inline Span span_of(const Batch& b, int64_t u) {
  if (!b.off) return Span{0, b.steps};
  const int64_t lo = b.off[u], n = b.off[u + 1] - lo;
  return b.steps ? Span{0, n < b.steps ? n : b.steps} : Span{lo, n};
}
// ---- the division of a batch over threads ----------------------------------------------------------
// A workgroup owns `seqs` sequences and `cb` groups of V neighbouring columns; its threads are (time slot, column group)
// pairs, `per` slots to a sequence.  A tile is per * R rows: a thread keeps the R x V values of its slot in registers,
// leaves the composition of its rows in LDS, and after one barrier composes those of the slots before it onto the state
// that enters the tile, then walks its rows from there: every value is read and written once.  A wave's load is cb * V
// neighbouring values of a row (and of the next slot's row).
constexpr int kSeqThreads = 512;
constexpr int kSlotRows = 8;   // R: composing costs per / R steps a value, registers 2 .. 6 R V

// Where the sequences and columns are too few for the card, a sequence is also cut into `pieces` of `piece_tiles` tiles, a
// workgroup each: a first kernel composes every piece into one entry of a workspace, the second one composes the entries before its
// piece and goes on from there. The rows are read twice; a single pass would have each workgroup hold its rows while it waits for
// the entries of all before it.
struct Split {
  int32_t groups, cb;    // column groups of a row, of a workgroup
  int32_t column_blocks; // workgroups to a row
  int32_t blocks;        // workgroups to a column block
  int32_t seqs, per;     // sequences of a workgroup, time slots of a sequence
  int32_t pieces, piece_tiles;  // pieces > 1 only with seqs == 1
  int32_t near;          // the rows of a tile lie within 4 GiB in every array
};

// V neighbouring values of a row; AL: rows are aligned to all of them, one access.
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T v[V];
};
template <bool AL, typename T, int V>
__device__ inline void load_pack(Pack<T, V>& r, const T* p) {
  if constexpr (AL || V == 1) {
    r = *(const Pack<T, V>*)p;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = p[i];
  }
}
// The one rounding to the type of the rows: everything before it is 32 or 64 bits wide.
template <bool AL, int V, typename T>
__device__ inline void store_pack(T* p, const float* f) {
  if constexpr (AL || V == 1) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)f[i];
    *(Pack<T, V>*)p = r;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = (T)f[i];
  }
}

// A value that all lanes agree on, in scalar registers.
__device__ inline int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline int64_t scalar(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)scalar((int)v) | (uint64_t)(uint32_t)scalar((int)(v >> 32)) << 32);
}

// What a thread works on.  Threads behind the last slot or column group are doubles of others: in full tiles they compute and
// write the same values, so that no access to rows needs a predicate. (y may be x: what a thread leaves in LDS before the barrier
// depends on all rows it has loaded, and rows are written behind the barrier.) Elsewhere only owners write.
struct Seat {
  int64_t u;           // sequence
  Span s;
  int n, sub, slot, cg, col;
  int wide;            // column groups that the workgroup has: the last block of a row may have fewer than the others
  int piece, tile, tiles, full;  // the tiles [tile, tiles) of the sequence, those below `full` without a missing row
  bool on;             // there is such a sequence
  bool there;          // the workgroup has something to do
  bool own;            // not a double
};
template <int V>
__device__ inline Seat seat_of(const Batch& b, const Split& w) {
  Seat t;
  // Workgroups go to the 8 XCDs in turn: the column blocks of the same rows are 8 apart, so that they run on one
  // XCD at about the same time and share the cache lines at their borders (2048 x 512 rows of 257 floats: 2270 -> 4500 GB/s).
  const int eight = blockIdx.x / (8 * w.column_blocks), r = blockIdx.x - eight * 8 * w.column_blocks;
  const int column_block = r / 8, at = eight * 8 + r % 8, block = at / w.pieces;
  t.there = at < w.blocks;
  t.piece = at - block * w.pieces;
  t.slot = threadIdx.x / w.cb;
  t.cg = (int)threadIdx.x - t.slot * w.cb;
  t.wide = min(w.groups - column_block * w.cb, w.cb);
  t.own = t.slot < w.seqs * w.per && t.cg < t.wide;
  t.cg = min(t.cg, t.wide - 1);
  if (t.slot >= w.seqs * w.per) t.slot = 0;
  t.col = (column_block * w.cb + t.cg) * V;
  const int tile_rows = w.per * kSlotRows;
  if (w.seqs > 1) {     // several sequences of one tile
    const int g = t.slot / w.per;
    t.sub = t.slot - g * w.per;
    t.u = (int64_t)block * w.seqs + g;
    t.on = t.u < b.n_seq;
    t.s = t.on ? span_of(b, t.u) : Span{0, 0};
    t.n = (int)t.s.n;
    t.tile = 0, t.tiles = 1, t.full = 0;
  } else {              // one sequence: everything but sub and the columns is the same for all threads, in scalar registers
    t.sub = t.slot;
    t.on = t.there;
    t.u = t.there ? b.order ? b.order[block] : block : 0;
    t.s = span_of(b, t.u);
    t.n = (int)t.s.n;
    t.tile = t.piece * w.piece_tiles;
    t.tiles = min((t.n + tile_rows - 1) / tile_rows, t.tile + w.piece_tiles);
    t.full = w.near ? max(min(t.n / tile_rows, t.tiles), t.tile) : t.tile;
  }
  t.tile = scalar(t.tile), t.tiles = scalar(t.tiles), t.full = scalar(t.full);
  return t;
}

// Rows of one sequence in any order of visit.  Full tiles: the address is a base that all threads share (scalar registers)
// plus 32 bits of the thread that never change, so a row costs no vector arithmetic.  Otherwise rows behind the end
// repeat the last one, and a thread without rows reads the first row of the array (a batch without any rows has null
// arrays, and nothing is read).  No branch in either form, so that the loads of the next tile go out while the
// current one is worked on; loads behind a store would have to wait for it (vmcnt counts both in order).
template <typename T>
struct Lane {
  const T* p;            // row 0 of the visit, the thread's column
  int64_t rs;            // to the next row of the visit
  const char* base;      // lowest row of tile 0, column 0
  int64_t tile_step, row_step;   // bytes
  uint32_t off;
};
template <int V, typename T>
__device__ inline Lane<T> lane_of(const Rows<T>& r, const Batch& b, const Split& w, const Seat& t) {
  Lane<T> f;
  const int64_t first = (b.steps ? t.u * r.ss : 0) + (t.s.first + (b.reverse ? t.n - 1 : 0)) * r.rs;
  f.rs = t.n == 0 ? 0 : b.reverse ? -r.rs : r.rs;
  f.p = r.p + (t.n == 0 ? 0 : first + t.col);
  // slots of a tile upwards in memory: the last one comes first in reverse (used where a workgroup has one sequence)
  f.base = (const char*)(r.p + scalar(first - (b.reverse ? (int64_t)(w.per - 1) * kSlotRows * r.rs : 0)));
  f.row_step = (b.reverse ? -r.rs : r.rs) * (int64_t)sizeof(T);
  f.tile_step = f.row_step * (w.per * kSlotRows);
  f.off = ((b.reverse ? w.per - 1 - t.sub : t.sub) * kSlotRows * (uint32_t)r.rs + t.col) * (uint32_t)sizeof(T);
  return f;
}
// The thread's offset, opaque, so that its extension to 64 bits stays next to the access: scalar base + 32-bit vector offset is
// one addressing mode, and out of a loop the compiler would add them with vector instructions instead.
__device__ inline uint32_t here(uint32_t off) {
#ifdef __HIP__   // a host build has no such register
  asm("" : "+v"(off));
#endif
  return off;
}
template <bool FULL, bool AL, typename T, typename S, int V>
__device__ inline void load_rows(Pack<T, V> (&r)[kSlotRows], const Lane<S>& f, const Seat& t, const Split& w, int tile) {
  if constexpr (FULL) {
    const char* p = f.base + tile * f.tile_step;
    const uint32_t off = here(f.off);
#pragma unroll
    for (int i = 0; i < kSlotRows; ++i, p += f.row_step) load_pack<AL>(r[i], (const T*)(p + off));
  } else {
    const int t0 = (tile * w.per + t.sub) * kSlotRows, last = max(t.n - 1, 0);
    const T* p = f.p + min(t0, last) * f.rs;
#pragma unroll
    for (int i = 0; i < kSlotRows; ++i) {
      load_pack<AL>(r[i], p);
      p += t0 + i < last ? f.rs : 0;
    }
  }
}
// Where row r of the thread's slot goes (off: its offset, here()).
template <bool FULL, typename T>
__device__ inline T* row_at(const Lane<T>& f, const Seat& t, const Split& w, int tile, int r, uint32_t off) {
  if constexpr (FULL) return (T*)(f.base + tile * f.tile_step + r * f.row_step + off);
  return (T*)f.p + ((tile * w.per + t.sub) * kSlotRows + r) * f.rs;
}

template <bool AL, int V, typename T>
__device__ inline void zero_behind(const Rows<T>& y, const Batch& b, const Split& w, const Seat& t) {
  const float z[V] = {};
  for (int64_t r = t.n + t.piece * w.per + t.sub; r < b.steps; r += w.pieces * w.per) store_pack<AL, V>(y.p + t.u * y.ss + r * y.rs + t.col, z);
}

// The rows of a slot's run of a piece: `run` neighbouring rows from row `begin` on, R at a time.
template <typename T>
struct RunLane {
  Lane<T> f;
  const char* base;
  uint32_t off;
};
template <typename T>
__device__ inline RunLane<T> run_of(const Lane<T>& f, const Rows<T>& r, const Batch& b, const Split& w, const Seat& t, int run) {
  RunLane<T> l{f, nullptr, 0};
  const int64_t back = b.reverse ? (int64_t)(w.per - 1) * r.rs * sizeof(T) : 0;   // the last slot is the lowest one in reverse
  l.base = f.base + t.tile * f.tile_step + kSlotRows * back - run * back;
  l.off = ((b.reverse ? w.per - 1 - t.sub : t.sub) * run * (uint32_t)r.rs + t.col) * (uint32_t)sizeof(T);
  return l;
}
template <bool FULL, bool AL, typename T, typename S, int V>
__device__ inline void load_run(Pack<T, V> (&r)[kSlotRows], const RunLane<S>& l, const Seat& t, int begin, int at) {
  if constexpr (FULL) {
    const char* p = l.base + at * l.f.row_step;
    const uint32_t off = here(l.off);
#pragma unroll
    for (int i = 0; i < kSlotRows; ++i, p += l.f.row_step) load_pack<AL>(r[i], (const T*)(p + off));
  } else {
    const T* p = l.f.p + min(begin + at, t.n - 1) * l.f.rs;
#pragma unroll
    for (int i = 0; i < kSlotRows; ++i) {
      load_pack<AL>(r[i], p);
      p += begin + at + i < t.n - 1 ? l.f.rs : 0;
    }
  }
}

// ---- gated recurrence -----------------------------------------------------------------------------
// h_t = a_t h_{t-1} + b_t is a composition of maps h -> A h + X: a run of rows is one such map, and maps of neighbouring
// runs join to (A2 A1, A2 X1 + X2).  Bound: HBM, 3 values moved a value forward and 5 backward.  512 sequences of 1024 rows of 512
// bfloat16: forward 5.1 TB/s, backward 4.9 (a copy of that size 5.3); 10000 of 300 rows of 39 floats 5.4 and 5.1; 2048 of 512 rows of
// 257 floats 4.4 and 4.0 (column blocks share cache lines).  A batch of 64 sequences of 100 to 1500 rows of 1024 bfloat16
// 86 + 125 us, 4.1 TB/s: at the end the tiles of the longest ones follow each other with the card half empty.

// a = 1 / (1 + e) and 1 - a = e a from e = exp(-g), neither by a difference.  g is held above -87 so that e stays finite (a is
// 2^-125 there; a NaN stays one).  The hardware exponential and reciprocal are good to one unit in the last place, and the
// product with log2(e) adds |g| 2^-24.
__device__ inline void sigmoid2(float g, float& a, float& na) {
  const float e = __expf(-(g < -87.0f ? -87.0f : g));
  a = __builtin_amdgcn_rcpf(1.0f + e);
  na = e * a;
}

// The map of many rows, h -> m 2^e h + x.  The product of gates leaves the range of 32 bits long before the states do (0.5 to the power of
// 150), and 0 times an infinite state, or an infinite product times 0, is no state: the product is kept as mantissa and exponent, and
// a state is multiplied by one, then shifted by the other. m is 0 where a gate was 0, otherwise 0.5 <= |m| < 1, so that 100 of them
// may be multiplied before the next normalised(). Two long bfloat16 training sequences (60000 and 47001 rows of 384) 225 us; the plain
// product in 32 bits 222; in 64 bits, held between two bounds at every step of the chains below, 231.
struct alignas(16) ScanMap {
  float m;
  int e;
  float x;
};
__device__ inline ScanMap normalised(float m, int e, float x) {
  const int far = 1 << 20;   // shifts any state of 32 bits to 0 or infinity; sums of exponents stay inside 32 bits
  return ScanMap{__builtin_amdgcn_frexp_mantf(m), max(min(e + __builtin_amdgcn_frexp_expf(m), far), -far), x};
}
__device__ inline float mapped(const ScanMap& f, float h) { return __builtin_amdgcn_ldexpf(f.m * h, f.e) + f.x; }
// f, then e
__device__ inline ScanMap compose(const ScanMap& e, const ScanMap& f) { return ScanMap{e.m * f.m, e.e + f.e, mapped(e, f.x)}; }

struct ScanPtrs {
  const float *h0, *glast;
  float *last, *ckpt, *gh0;
  ScanMap* maps;   // [sequence][piece][column] where sequences are cut into pieces
};

// Checkpoint of (sequence, tile): float32 states that enter a tile.  Packed sequences get rows / K + u as their first one:
// at least as far apart as ceil(n / K).
__device__ inline int64_t checkpoint_row(const Batch& b, const Seat& t, int tile_rows) {
  return b.steps ? t.u * ((b.steps + tile_rows - 1) / tile_rows) : t.s.first / tile_rows + t.u;
}

template <typename T, int V>
struct ScanRows {
  Pack<T, V> x[kSlotRows], g[kSlotRows];
};

// The map of every piece: forward h -> A h + X from (x, gate), backward e -> A e + E from (gate, grad_y). A slot takes a contiguous
// run of the piece, so that the threads meet once.  Bound: HBM, 2 values read a value; 360000 rows of 256 float16: both kernels
// 209 us for 921 MB, 4.4 TB/s (whole, without pieces: 9.6 ms).
template <typename T, int V, bool AL, bool SIG, bool BACK>
__global__ void __launch_bounds__(kSeqThreads, 4) gated_scan_pieces_kernel(const Batch b, const Split w, const Rows<const T> x,
                                                                           const Rows<const T> g, const ScanPtrs q) {
  constexpr int R = kSlotRows;
  __shared__ ScanMap maps[kSeqThreads * V];
  const Seat t = seat_of<V>(b, w);
  if (!t.there || t.tile >= t.tiles || !g.p) return;   // the same for the whole workgroup
  const bool no_gy = BACK && !x.p;
  const int run = w.piece_tiles * R, piece = t.tile * w.per * R, first = piece + t.sub * run;
  const RunLane<const T> fg = run_of(lane_of<V>(g, b, w, t), g, b, w, t, run);
  const RunLane<const T> fx = no_gy ? fg : run_of(lane_of<V>(x, b, w, t), x, b, w, t, run);
  ScanMap A[V];
  float X[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = ScanMap{1.0f, 0, 0.0f}, X[v] = 0.0f;
  auto walk = [&](auto full) {
    constexpr bool FULL = full();
    const int len = FULL ? run : min(max(t.n - first, 0), run), last = BACK ? (len + R - 1) / R * R - R : 0;
    auto load = [&](ScanRows<T, V>& r, int at) {
      load_run<FULL, AL>(r.x, fx, t, first, at);
      load_run<FULL, AL>(r.g, fg, t, first, at);
    };
    ScanRows<T, V> in, next;
    load(in, last);
    for (int i = 0; i < len; i += R) {
      const int at = BACK ? last - i : i, k = len - at;
      load(next, BACK ? max(at - R, 0) : FULL ? min(at + R, run - R) : at + R);
      float P[V];
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 1.0f;
#pragma unroll
      for (int j = 0; j < R; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int r = BACK ? R - 1 - j : j;
          float a = (float)in.g[r].v[v], na = 1.0f;
          if constexpr (SIG) sigmoid2(a, a, na);
          const float xv = no_gy ? 0.0f : (float)in.x[r].v[v];
          const float nx = BACK ? a * (xv + X[v]) : fmaf(a, X[v], na * xv);
          X[v] = FULL || r < k ? nx : X[v];
          P[v] = FULL || r < k ? P[v] * a : P[v];
        }
#pragma unroll
      for (int v = 0; v < V; ++v) A[v] = normalised(A[v].m * P[v], A[v].e, 0.0f);
      in = next;
    }
  };
  if (w.near && piece + w.per * run <= t.n) walk(std::true_type());
  else walk(std::false_type());
#pragma unroll
  for (int v = 0; v < V; ++v) maps[(t.slot * V + v) * w.cb + t.cg] = ScanMap{A[v].m, A[v].e, X[v]};
  __syncthreads();
  if (t.sub == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      ScanMap f{1.0f, 0, 0.0f};
      for (int s = 0; s < w.per; ++s) f = compose(maps[((BACK ? w.per - 1 - s : s) * V + v) * w.cb + t.cg], f);
      q.maps[(t.u * w.pieces + t.piece) * b.ncol + t.col + v] = normalised(f.m, f.e, f.x);
    }
  }
}

// What enters a piece: the maps of the `count` pieces on the way to it, in order, on the state `h`.  Each slot composes a run of them,
// the slots meet in LDS.  `base` is the first map, `step` the distance to the next.
template <int V>
__device__ inline void enter_piece(float (&h)[V], const ScanMap* base, int64_t step, int count, const Split& w, const Seat& t, ScanMap* maps) {
  if (count == 0) return;
  const int run = (count + w.per - 1) / w.per, lo = t.sub * run, hi = min(lo + run, count);
  ScanMap f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = ScanMap{1.0f, 0, 0.0f};
  const ScanMap* p = base + lo * step;
#pragma unroll 8
  for (int i = lo; i < hi; ++i, p += step)
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = compose(p[v], f[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) maps[(t.slot * V + v) * w.cb + t.cg] = normalised(f[v].m, f[v].e, f[v].x);
  __syncthreads();
  for (int s = 0; s < w.per; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = mapped(maps[(s * V + v) * w.cb + t.cg], h[v]);
  __syncthreads();
}

template <typename T, int V, bool AL, bool SIG>
__global__ void __launch_bounds__(kSeqThreads, 4) gated_scan_kernel(const Batch b, const Split w, const Rows<const T> x, const Rows<const T> g,
                                                                    const Rows<T> y, const ScanPtrs q) {
  constexpr int R = kSlotRows;
  alignas(16) __shared__ float2 maps[2][kSeqThreads * V];   // of tiles in turn; all of it for the ScanMaps on the way to a piece
  const Seat t = seat_of<V>(b, w);
  if (!t.there) return;
  const Lane<const T> fx = lane_of<V>(x, b, w, t), fg = lane_of<V>(g, b, w, t);
  const Lane<T> fy = lane_of<V>(y, b, w, t);
  const int64_t end = t.u * b.ncol + t.col;   // of the states of a sequence
  float carry[V] = {}, h[V] = {};
  if (t.on && q.h0)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = q.h0[end + v];
  float* const ck = q.ckpt ? q.ckpt + checkpoint_row(b, t, w.per * R) * b.ncol + t.col : nullptr;

  auto work = [&](auto full, const ScanRows<T, V>& in, int tile) {
    constexpr bool FULL = full();
    const int k = FULL ? R : min(max(t.n - (tile * w.per + t.sub) * R, 0), R);
    float a[R][V], x1[R][V], A[V], X[V];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float av = (float)in.g[r].v[v], bv = (float)in.x[r].v[v];
        if constexpr (SIG) {
          float na;
          sigmoid2(av, av, na);
          bv *= na;
        }
        a[r][v] = FULL || r < k ? av : 1.0f;   // rows behind the end leave the state alone
        x1[r][v] = FULL || r < k ? bv : 0.0f;
        X[v] = r ? fmaf(a[r][v], X[v], x1[r][v]) : x1[r][v];
        A[v] = r ? A[v] * a[r][v] : a[r][v];
      }
    if (w.per > 1) {
      float2* const m = maps[tile & 1];
#pragma unroll
      for (int v = 0; v < V; ++v) m[(t.slot * V + v) * w.cb + t.cg] = make_float2(A[v], X[v]);
      __syncthreads();
      const float2* e = m + (t.slot - t.sub) * V * w.cb + t.cg;
#pragma unroll 4
      for (int s = 0; s < w.per; ++s, e += V * w.cb)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 f = e[v * w.cb];
          h[v] = s == t.sub ? carry[v] : h[v];
          carry[v] = fmaf(f.x, carry[v], f.y);
        }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = carry[v], carry[v] = fmaf(A[v], carry[v], X[v]);
    }
    if (ck && t.own && t.sub == 0 && k > 0)
#pragma unroll
      for (int v = 0; v < V; ++v) ck[(int64_t)tile * b.ncol + v] = h[v];
    const uint32_t to = here(fy.off);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = fmaf(a[r][v], h[v], x1[r][v]);
      if (FULL || (t.own && r < k)) store_pack<AL, V>(row_at<FULL>(fy, t, w, tile, r, to), h);
    }
  };

  if (x.p && t.tile < t.tiles) {   // the same for the whole workgroup
    ScanRows<T, V> in, next;
    auto load = [&](auto full, ScanRows<T, V>& r, int tile) {
      load_rows<full(), AL>(r.x, fx, t, w, tile);
      load_rows<full(), AL>(r.g, fg, t, w, tile);
    };
    int tile = t.tile;
    load(std::false_type(), in, tile);
    if (t.piece > 0) enter_piece(carry, q.maps + t.u * w.pieces * b.ncol + t.col, b.ncol, t.piece, w, t, (ScanMap*)maps);
    for (; tile + 1 < t.full; ++tile) {
      load(std::true_type(), next, tile + 1);
      work(std::true_type(), in, tile);
      in = next;
    }
    if (tile < t.full) {
      if (t.full < t.tiles) load(std::false_type(), next, t.full);
      work(std::true_type(), in, tile++);
      in = next;
    }
    for (; tile < t.tiles; ++tile) {   // at most once, unless rows lie far apart
      if (tile > t.full) load(std::false_type(), in, tile);
      work(std::false_type(), in, tile);
    }
  }
  // the state behind the last row, from the thread that walked it: the very value that y rounds
  const int lead = t.n > 0 ? (t.n - 1) / R % w.per : 0;
  if (t.on && t.own && q.last && t.sub == lead && (t.n > 0 ? t.tile < t.tiles && t.tiles * w.per * R >= t.n : t.piece == 0))
#pragma unroll
    for (int v = 0; v < V; ++v) q.last[end + v] = t.n > 0 ? h[v] : carry[v];
  if (t.on && t.own && b.steps) zero_behind<AL, V>(y, b, w, t);
}

// Gradient.  With e_t = a_t delta_t, delta_t = gy_t + e_{t+1}, the way back is a composition of maps e -> A (gy + e) with the
// same products of gates, from the last tile to the first; the states h_{t-1} that dgate needs are walked
// again from the checkpoint of the tile.
// 152 to 197 registers of V = 2 leave 2 waves a SIMD; bounded to 128 they spill, and the step on 64 x 1500 x 1024 takes 510 us
// instead of 213.
template <typename T, int V>
struct ScanGradRows {
  Pack<T, V> x[kSlotRows], g[kSlotRows], d[kSlotRows];
  Pack<float, V> h;   // the state that enters the tile
};

template <typename T, int V, bool AL, bool SIG>
__global__ void __launch_bounds__(kSeqThreads, 2) gated_scan_backward_kernel(const Batch b, const Split w, const Rows<const T> x,
                                                                             const Rows<const T> g, const Rows<const T> gy, const Rows<T> gx,
                                                                             const Rows<T> gg, const ScanPtrs q) {
  constexpr int R = kSlotRows;
  alignas(16) __shared__ float maps[2][3][kSeqThreads * V];
  const Seat t = seat_of<V>(b, w);
  if (!t.there) return;
  const bool no_gy = !gy.p;
  const Lane<const T> fx = lane_of<V>(x, b, w, t), fg = lane_of<V>(g, b, w, t), fd = no_gy ? fx : lane_of<V>(gy, b, w, t);
  const Lane<T> fgx = lane_of<V>(gx, b, w, t), fgg = lane_of<V>(gg, b, w, t);
  const int64_t end = t.u * b.ncol + t.col;
  float carry[V] = {};
  if (t.on && q.glast)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = q.glast[end + v];
  const int64_t ck_step = t.n > 0 ? b.ncol : 0;
  const float* const ck = t.n > 0 ? q.ckpt + checkpoint_row(b, t, w.per * R) * b.ncol + t.col : q.ckpt;

  auto load = [&](auto full, ScanGradRows<T, V>& r, int tile) {
    load_rows<full(), AL>(r.x, fx, t, w, tile);
    load_rows<full(), AL>(r.g, fg, t, w, tile);
    load_rows<full(), AL>(r.d, fd, t, w, tile);
    load_pack<false>(r.h, ck + tile * ck_step);
  };
  auto work = [&](auto full, const ScanGradRows<T, V>& in, int tile) {
    constexpr bool FULL = full();
    const int k = FULL ? R : min(max(t.n - (tile * w.per + t.sub) * R, 0), R);
    float a[R][V], na[R][V], A[V], X[V], E[V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.0f, X[v] = 0.0f, E[v] = 0.0f, h[v] = in.h.v[v];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float av = (float)in.g[r].v[v], nv = 1.0f;
        if constexpr (SIG) sigmoid2(av, av, nv);
        a[r][v] = FULL || r < k ? av : 1.0f;
        na[r][v] = nv;
        X[v] = fmaf(a[r][v], X[v], FULL || r < k ? nv * (float)in.x[r].v[v] : 0.0f);
        A[v] *= a[r][v];
      }
    auto delta = [&](int r, int v, float e) { return ((FULL || r < k) && !no_gy ? (float)in.d[r].v[v] : 0.0f) + e; };
#pragma unroll
    for (int r = R - 1; r >= 0; --r)
#pragma unroll
      for (int v = 0; v < V; ++v) E[v] = a[r][v] * delta(r, v, E[v]);
    float e[V];
    if (w.per > 1) {
      float(*const m)[kSeqThreads * V] = maps[tile & 1];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = (t.slot * V + v) * w.cb + t.cg;
        m[0][i] = A[v], m[1][i] = X[v], m[2][i] = E[v];
      }
      __syncthreads();
      const int first = (t.slot - t.sub) * V * w.cb + t.cg;
#pragma unroll 2
      for (int s = 0; s < w.per; ++s)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int i = first + (s * V + v) * w.cb, j = first + ((w.per - 1 - s) * V + v) * w.cb;
          h[v] = s < t.sub ? fmaf(m[0][i], h[v], m[1][i]) : h[v];
          e[v] = w.per - 1 - s == t.sub ? carry[v] : e[v];
          carry[v] = fmaf(m[0][j], carry[v], m[2][j]);
        }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) e[v] = carry[v], carry[v] = fmaf(A[v], carry[v], E[v]);
    }
    if (FULL || k > 0) {
      float hp[R][V];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          hp[r][v] = h[v];
          h[v] = fmaf(a[r][v], h[v], FULL || r < k ? na[r][v] * (float)in.x[r].v[v] : 0.0f);
        }
      const uint32_t to_x = here(fgx.off), to_g = here(fgg.off);
#pragma unroll
      for (int r = R - 1; r >= 0; --r) {
        float dx[V], dg[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = delta(r, v, e[v]);
          dx[v] = SIG ? na[r][v] * d : d;
          e[v] = a[r][v] * d;
          dg[v] = SIG ? e[v] * na[r][v] * (hp[r][v] - (float)in.x[r].v[v]) : d * hp[r][v];
        }
        if (FULL || (t.own && r < k)) {
          store_pack<AL, V>(row_at<FULL>(fgx, t, w, tile, r, to_x), dx);
          store_pack<AL, V>(row_at<FULL>(fgg, t, w, tile, r, to_g), dg);
        }
      }
    }
  };

  if (x.p && t.tile < t.tiles) {   // the same for the whole workgroup
    ScanGradRows<T, V> in, next;
    if (w.pieces > 1) {
      const int piece_rows = w.piece_tiles * w.per * R, pieces = (t.n + piece_rows - 1) / piece_rows;   // of this sequence
      enter_piece(carry, q.maps + (t.u * w.pieces + pieces - 1) * b.ncol + t.col, -(int64_t)b.ncol, pieces - 1 - t.piece, w, t, (ScanMap*)maps);
    }
    int tile = t.tiles - 1;
    for (; tile >= t.full; --tile) {   // at most once, unless rows lie far apart
      load(std::false_type(), in, tile);
      work(std::false_type(), in, tile);
    }
    if (tile >= t.tile) {
      load(std::true_type(), in, tile);
      for (; tile > t.tile; --tile) {
        load(std::true_type(), next, tile - 1);
        work(std::true_type(), in, tile);
        in = next;
      }
      work(std::true_type(), in, tile);
    }
  }
  if (t.on && t.own && q.gh0 && t.sub == 0 && t.piece == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) q.gh0[end + v] = carry[v];
  if (t.on && t.own && b.steps) {
    zero_behind<AL, V>(gx, b, w, t);
    zero_behind<AL, V>(gg, b, w, t);
  }
}

// One step of live sequences, a thread to a value: 64 x 512 floats are 0.7 MB, the launch is what it costs (4.7 us each in a
// captured sequence of them).
template <typename T, bool SIG>
__global__ void __launch_bounds__(256) gated_scan_step_kernel(int64_t n, int ncol, const T* x, int64_t x_ld, const T* g, int64_t g_ld,
                                                              const float* hin, float* hout, T* y, int64_t y_ld) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * ncol) return;
  const int64_t u = i / ncol;
  const int c = (int)(i % ncol);
  float a = (float)g[u * g_ld + c], v = (float)x[u * x_ld + c];
  if constexpr (SIG) {
    float na;
    sigmoid2(a, a, na);
    v *= na;
  }
  const float h = fmaf(a, hin[i], v);
  hout[i] = h;
  y[u * y_ld + c] = (T)h;
}

// ---- running normalisation ---------------------------------------------------------------------------
// A run of k rows is (m, q): its mean and its sum of squared deviations under the weights decay^(k-1) .. 1, whose sum is
// g(k) = 1 + decay + .. + decay^(k-1). A run behind one of weight w joins to
//   w' = decay^k w + g,  f = g / w',  m' = m + (m_run - m) f,  q' = decay^k q + q_run + (m_run - m)^2 decay^k w f,
// without a difference of squares. The weights depend on the row number alone: they are carried in 64 bits from tile to tile (at the fixed
// point of w the roundings of 32 bits have one sign: 7e-6 of w off after 20000 rows at decay 0.995), and f and decay^k w f are
// computed once per slot. The mean that enters a tile is carried in 64 bits and the tile composes 32-bit deviations from it: a
// cumulative mean of n rows would otherwise collect sqrt(n) / 4 units in the last place.
// Bound: HBM, one value read and one written, closely followed by the vector pipe: 31 instructions a value in full tiles, 47 with the
// ends of 299 rows (68 % of the cycles of 10000 sequences of 39 columns: 228 us, 4.1 TB/s), so slots are few where sequences are
// many (every join is shared by R values only). One hour of 39 columns, cumulative: 12 us for the pieces, 33 us for the rows.
struct NormArgs {
  double decay, log_decay;      // log_decay = log1p(decay - 1)
  // decay^k and g(k) of a slot, a tile, a slot's run of a piece, a piece
  double slot_decay, slot_grown, tile_decay, tile_grown, run_decay, run_grown, piece_decay, piece_grown;
  float eps, decayed[kSlotRows], grown[kSlotRows], inv_grown[kSlotRows];   // decay^k, g(k), 1 / g(k) for k = 1 .. R
  int center_only;
  const float* state_in;
  float* state_out;
  float2* runs;                 // [sequence][piece][column] (m, q) where sequences are cut into pieces
};

// decay^k and g(k)
__device__ inline void weights_of(const NormArgs& a, double k, double& decayed, double& grown) {
  const double em = expm1(k * a.log_decay);
  decayed = 1.0 + em;
  grown = a.decay == 1.0 ? k : em / (a.decay - 1.0);
}

// (m, q) of k rows, one after the other.
template <int V, int N, bool ALL>
__device__ inline void norm_run(float (&m)[V], float (&q)[V], float& w, float decay, const Pack<float, V> (&x)[N], int k, const float* inv) {
#pragma unroll
  for (int r = 0; r < N; ++r) {
    w = ALL || r < k ? fmaf(decay, w, 1.0f) : w;
    const float f = inv ? inv[r] : __builtin_amdgcn_rcpf(w);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float d = x[r].v[v] - m[v], mn = fmaf(d, f, m[v]), qn = fmaf(d, x[r].v[v] - mn, decay * q[v]);
      m[v] = ALL || r < k ? mn : m[v];
      q[v] = ALL || r < k ? qn : q[v];
    }
  }
}

// (w, m, q) and behind it (g, m2, q2) after `decayed` of the first is left.
__device__ inline void norm_join(float& w, float& m, float& q, float decayed, float g, float m2, float q2) {
  const float old = decayed * w, sum = old + g, f = old > 0.0f ? g * __builtin_amdgcn_rcpf(sum) : 1.0f, d = m2 - m;   // g > 0
  w = sum;
  m = fmaf(d, f, m);
  q = fmaf(decayed, q, fmaf(d * d, old * f, q2));
}

template <int V, bool AL>
__global__ void __launch_bounds__(kSeqThreads, 4) running_norm_pieces_kernel(const Batch b, const Split w, const Rows<const float> x, const NormArgs a) {
  constexpr int R = kSlotRows;
  __shared__ float2 runs[kSeqThreads * V];
  const Seat t = seat_of<V>(b, w);
  if (!t.there || t.tile >= t.tiles || !x.p) return;   // the same for the whole workgroup
  const int run = w.piece_tiles * R, first = t.tile * w.per * R, begin = first + t.sub * run;
  const RunLane<const float> fx = run_of(lane_of<V>(x, b, w, t), x, b, w, t, run);
  float m[V] = {}, q[V] = {};
  auto walk = [&](auto full) {
    constexpr bool FULL = full();
    const int len = FULL ? run : min(max(t.n - begin, 0), run);
    float sum = 0.0f;
    Pack<float, V> in[R], next[R];
    load_run<FULL, AL>(in, fx, t, begin, 0);
    for (int i = 0; i < len; i += R) {
      load_run<FULL, AL>(next, fx, t, begin, FULL ? min(i + R, run - R) : i + R);
      norm_run<V, R, FULL>(m, q, sum, (float)a.decay, in, len - i, nullptr);
#pragma unroll
      for (int r = 0; r < R; ++r) in[r] = next[r];
    }
  };
  if (w.near && first + w.per * run <= t.n) walk(std::true_type());
  else walk(std::false_type());
#pragma unroll
  for (int v = 0; v < V; ++v) runs[(t.slot * V + v) * w.cb + t.cg] = make_float2(m[v], q[v]);
  __syncthreads();
  if (t.sub == 0) {
    double l = a.run_decay, g = a.run_grown;
    float ws = 0.0f, ms[V] = {}, qs[V] = {};
    for (int s = 0; s < w.per; ++s) {
      const int k = min(max(t.n - first - s * run, 0), run);
      if (k == 0) break;
      if (k < run) weights_of(a, k, l, g);
      float wn = ws;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 e = runs[(s * V + v) * w.cb + t.cg];
        wn = ws;
        norm_join(wn, ms[v], qs[v], (float)l, (float)g, e.x, e.y);
      }
      ws = wn;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) a.runs[(t.u * w.pieces + t.piece) * b.ncol + t.col + v] = make_float2(ms[v], qs[v]);
  }
}

// 1 / sqrt(v).  The hardware's takes a subnormal for 0. BARE: an eps that does not keep the variance out of the subnormals alone; a kernel
// of its own, as a choice within costs every batch 3 % (10000 sequences of 299 rows of 39: 215 -> 222 us).
template <bool BARE>
__device__ inline float inverse_root(float v) {
  const bool lift = BARE && v < 0x1p-126f;
  const float r = __builtin_amdgcn_rsqf(lift ? v * 0x1p64f : v);
  return lift ? r * 0x1p32f : r;
}

template <typename T, int V, bool AL, bool BARE>
__global__ void __launch_bounds__(kSeqThreads, 4) running_norm_kernel(const Batch b, const Split w, const Rows<const float> x, const Rows<T> y,
                                                                      const NormArgs a) {
  constexpr int R = kSlotRows;
  // twice, for tiles in turn: the run of every (slot, column); of every slot the weights of its join, (f, decay^k w f, decay^k, -), and
  // 1 / w of its rows
  extern __shared__ float4 shared[];
  const Seat t = seat_of<V>(b, w);
  if (!t.there) return;
  const int slots = w.seqs * w.per;
  float4* const joins = shared;
  float4* const inverses = joins + 2 * slots;
  float2* const runs = (float2*)(inverses + 2 * slots * (R / 4));
  const Lane<const float> fx = lane_of<V>(x, b, w, t);
  const Lane<T> fy = lane_of<V>(y, b, w, t);
  const float decay = (float)a.decay;
  const int64_t state = t.u * (1 + 2 * (int64_t)b.ncol);
  // decay^k and g(k) of the rows of a tile before the thread's slot
  double before_decay = 1.0, before_grown = 0.0;
  for (int s = 0; s < t.sub; ++s) before_decay *= a.slot_decay, before_grown = fma(a.slot_decay, before_grown, a.slot_grown);
  const float own_decayed = a.decayed[min(t.cg, R - 1)], own_grown = a.grown[min(t.cg, R - 1)];   // read here: a load in the loop waits for all others
  double weight = 0.0, mean[V] = {};   // that enter the tile
  float square[V] = {}, m[V] = {}, q[V] = {}, last_weight = 0.0f;
  if (t.on && a.state_in) {
    weight = a.state_in[state];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // beside a weight of 0 the first row is the mean, whatever the state's was: a step from there would leave a rounding of the way between
      // them, of either sign, where s has the product with that way added
      mean[v] = weight < 0x1p-22 ? 0.0 : a.state_in[state + 1 + t.col + v];
      square[v] = a.state_in[state + 1 + b.ncol + t.col + v];
    }
  }

  auto work = [&](auto full, const Pack<float, V>(&in)[R], int tile) {
    constexpr bool FULL = full();
    const int k = FULL ? R : min(max(t.n - (tile * w.per + t.sub) * R, 0), R), turn = tile & 1;
    const float ws = (float)fma(before_decay, weight, before_grown);
    last_weight = fmaf(FULL || k == R ? a.decayed[R - 1] : k > 0 ? a.decayed[k - 1] : 1.0f, ws, FULL || k == R ? a.grown[R - 1] : k > 0 ? a.grown[k - 1] : 0.0f);
    float base[V], off[V];
#pragma unroll
    for (int v = 0; v < V; ++v) base[v] = (float)mean[v], off[v] = (float)(mean[v] - base[v]);
    float4* const inv = inverses + (turn * slots + t.slot) * (R / 4);
    // 1 / w of the rows: the column groups that there are take one row each, and further ones where they are fewer than the rows
    if (t.cg < R) ((float*)inv)[t.cg] = __builtin_amdgcn_rcpf(fmaf(own_decayed, ws, own_grown));
    for (int r = t.cg + t.wide; r < R; r += t.wide) ((float*)inv)[r] = __builtin_amdgcn_rcpf(fmaf(a.decayed[r], ws, a.grown[r]));
    if (w.per > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = 0.0f, q[v] = 0.0f;
      float none = 0.0f;
      norm_run<V, R, FULL>(m, q, none, decay, in, k, a.inv_grown);
      float4* const j = joins + turn * slots;
      float2* const e = runs + turn * slots * V * w.cb + t.cg;
#pragma unroll
      for (int v = 0; v < V; ++v) e[(t.slot * V + v) * w.cb] = make_float2(m[v] - base[v], q[v]);
      if (t.cg == 0) {
        const float l = FULL || k == R ? a.decayed[R - 1] : k > 0 ? a.decayed[k - 1] : 1.0f;
        const float g = FULL || k == R ? a.grown[R - 1] : k > 0 ? a.grown[k - 1] : 0.0f;
        const float old = l * ws, f = g == 0.0f ? 0.0f : old > 0.0f ? g * __builtin_amdgcn_rcpf(old + g) : 1.0f;   // a first run is its own mean
        j[t.slot] = make_float4(f, old * f, l, 0.0f);
      }
      __syncthreads();
      const float2* r = e + (t.slot - t.sub) * V * w.cb;
      const float4* p = j + (t.slot - t.sub);
      auto join = [&]() {
        const float4 h = *p++;
#pragma unroll
        for (int v = 0; v < V; ++v, r += w.cb) {
          const float2 run = *r;
          const float d = run.x - off[v];
          off[v] = fmaf(d, h.x, off[v]);
          square[v] = fmaf(h.z, square[v], fmaf(d * d, h.y, run.y));
        }
      };
      int i = 0;
#pragma unroll 4
      for (; i < t.sub; ++i) join();
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = base[v] + off[v], q[v] = square[v];
#pragma unroll 4
      for (; i < w.per; ++i) join();
#pragma unroll
      for (int v = 0; v < V; ++v) mean[v] = (double)base[v] + off[v];
      weight = fma(a.tile_decay, weight, a.tile_grown);   // behind a last tile with missing rows it is not used
    } else {
      __syncthreads();   // 1 / w
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = base[v], q[v] = square[v];
    }
    const uint32_t to = here(fy.off);
    float f[R];
#pragma unroll
    for (int r = 0; r < R; r += 4) {
      const float4 four = inv[r / 4];
      f[r] = four.x, f[r + 1] = four.y, f[r + 2] = four.z, f[r + 3] = four.w;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = in[r].v[v] - m[v], mn = fmaf(d, f[r], m[v]), c = in[r].v[v] - mn, qn = fmaf(d, c, decay * q[v]);
        o[v] = a.center_only ? c : c * inverse_root<BARE>(fmaf(qn, f[r], a.eps));
        m[v] = FULL || r < k ? mn : m[v];
        q[v] = FULL || r < k ? qn : q[v];
      }
      if (FULL || (t.own && r < k)) store_pack<AL, V>(row_at<FULL>(fy, t, w, tile, r, to), o);
    }
  };

  if (x.p && t.tile < t.tiles) {   // the same for the whole workgroup
    Pack<float, V> in[R], next[R];
    int tile = t.tile;
    load_rows<false, AL>(in, fx, t, w, tile);
    if (t.piece > 0) {
      // the pieces before this one, all of them full: each slot joins a run of them, the slots meet in LDS with the weights of
      // their runs in 64 bits. The means are joined as 32-bit deviations from the one that enters the sequence: below half a unit in the
      // last place of a deviation a run, one run a slot (at most 64), where the mean itself is rounded once at the end (in 64 bits the second
      // kernel of one hour of 39 columns takes 35.5 us instead of 33).
      const int run = (t.piece + w.per - 1) / w.per, lo = t.sub * run, hi = min(lo + run, t.piece);
      const float2* p = a.runs + (t.u * w.pieces + lo) * b.ncol + t.col;
      double run_decay = 1.0, run_grown = 0.0;
      float sum = 0.0f;
#pragma unroll 8
      for (int i = lo; i < hi; ++i, p += b.ncol) {
        float wn = sum;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          wn = sum;
          norm_join(wn, m[v], q[v], (float)a.piece_decay, (float)a.piece_grown, p[v].x, p[v].y);
        }
        sum = wn;
        run_decay *= a.piece_decay;
        run_grown = fma(a.piece_decay, run_grown, a.piece_grown);
      }
      double* const weights = (double*)joins;   // two of every slot
#pragma unroll
      for (int v = 0; v < V; ++v) runs[(t.slot * V + v) * w.cb + t.cg] = make_float2(m[v], q[v]);
      if (t.cg == 0) weights[2 * t.slot] = run_decay, weights[2 * t.slot + 1] = run_grown;
      __syncthreads();
      float off[V] = {}, base[V];
#pragma unroll
      for (int v = 0; v < V; ++v) base[v] = (float)mean[v], off[v] = (float)(mean[v] - base[v]);
      for (int s = 0; s < w.per && s * run < t.piece; ++s) {
        const double old = weights[2 * s] * weight, g = weights[2 * s + 1];
        const float l = (float)weights[2 * s], f = old > 0.0 ? (float)g * __builtin_amdgcn_rcpf((float)(old + g)) : 1.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float2 e = runs[(s * V + v) * w.cb + t.cg];
          const float d = e.x - base[v] - off[v];
          off[v] = fmaf(d, f, off[v]);
          square[v] = fmaf(l, square[v], fmaf(d * d, (float)old * f, e.y));
        }
        weight = old + g;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) mean[v] = (double)base[v] + off[v];
      __syncthreads();
    }
    for (; tile + 1 < t.full; ++tile) {
      load_rows<true, AL>(next, fx, t, w, tile + 1);
      work(std::true_type(), in, tile);
#pragma unroll
      for (int r = 0; r < R; ++r) in[r] = next[r];
    }
    if (tile < t.full) {
      if (t.full < t.tiles) load_rows<false, AL>(next, fx, t, w, t.full);
      work(std::true_type(), in, tile++);
#pragma unroll
      for (int r = 0; r < R; ++r) in[r] = next[r];
    }
    for (; tile < t.tiles; ++tile) {   // at most once, unless rows lie far apart
      if (tile > t.full) load_rows<false, AL>(in, fx, t, w, tile);
      work(std::false_type(), in, tile);
    }
  }
  // the state behind the last row, from the thread that walked it
  const int lead = t.n > 0 ? (t.n - 1) / R % w.per : 0;
  if (t.on && t.own && a.state_out && t.sub == lead && (t.n > 0 ? t.tile < t.tiles && t.tiles * w.per * R >= t.n : t.piece == 0)) {
    auto entered = [&](int64_t i) { return a.state_in ? a.state_in[state + i] : 0.0f; };   // passes through where there are no rows
    if (t.col == 0) a.state_out[state] = t.n > 0 ? last_weight : entered(0);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a.state_out[state + 1 + t.col + v] = t.n > 0 ? m[v] : entered(1 + t.col + v);
      a.state_out[state + 1 + b.ncol + t.col + v] = t.n > 0 ? q[v] : entered(1 + b.ncol + t.col + v);
    }
  }
  if (t.on && t.own && b.steps) zero_behind<AL, V>(y, b, w, t);
}

// ---- dropout --------------------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): two 32 x 32 -> 64 bit
// products a round, the key raised by two Weyl constants.
__device__ inline uint4 philox4x32_10(uint64_t block, uint64_t step, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}
// Bit k of the result: field k of the block is below the threshold, its element dropped.
__device__ inline uint32_t philox_dropped(uint64_t block, uint64_t step, uint64_t seed, uint32_t threshold) {
  const uint4 w = philox4x32_10(block, step, seed);
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) bits |= ((v[k] & 0xFFFFu) < threshold ? 1u : 0u) << (2 * k) | ((v[k] >> 16) < threshold ? 2u : 0u) << (2 * k);
  return bits;
}

struct Dropout {
  uint64_t seed, step;
  const int64_t* step_device;
  uint32_t threshold;
  float scale;
  __device__ uint64_t at() const { return step_device ? (uint64_t)*step_device : step; }
};

// per = element: a thread takes the 8 consecutive elements of one block. FLAT: rows back to back in both arrays and 16-byte
// aligned, an element is its number. Otherwise (row, column) of the first one by division, then step by step.
// Bound: HBM, read once and written once: 20000 x 4369 bfloat16 75 us a pass, 4.6 TB/s; the 20 wide products of a block are shared
// by 8 elements (an element to a thread: 290 us).
template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) dropout_element_kernel(const Batch b, int64_t n_rows, const Dropout d, const Rows<const T> x,
                                                              const Rows<T> y) {
  const int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x, total = n_rows * b.ncol, e0 = block * 8;
  if (e0 >= total) return;
  const uint32_t gone = philox_dropped((uint64_t)block, d.at(), d.seed, d.threshold);
  if (FLAT && e0 + 8 <= total) {
    constexpr int V = 16 / sizeof(T);
    Pack<T, V> r[8 / V];
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) r[i] = *(const Pack<T, V>*)(x.p + e0 + i * V);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      T& v = r[i / V].v[i % V];
      v = gone >> i & 1 ? (T)0.0f : (T)((float)v * d.scale);
    }
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) *(Pack<T, V>*)(y.p + e0 + i * V) = r[i];
    return;
  }
  const int64_t row = total < ((int64_t)1 << 32) ? (int64_t)((uint32_t)e0 / (uint32_t)b.ncol) : e0 / b.ncol;
  int64_t u = 0, t = row;
  if (b.steps) {
    u = n_rows < ((int64_t)1 << 32) ? (int64_t)((uint32_t)row / (uint32_t)b.steps) : row / b.steps;
    t = row - u * b.steps;
  }
  int c = (int)(e0 - row * b.ncol);
  const int k = (int)min((int64_t)8, total - e0);
  // all loads first; behind the last element they repeat it
  int64_t to[8];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = (float)x.p[u * x.ss + t * x.rs + c];
    to[i] = u * y.ss + t * y.rs + c;
    const bool more = i + 1 < k, wrap = more && c + 1 == b.ncol, next = wrap && t + 1 == b.steps;   // packed rows: steps is 0
    c = wrap ? 0 : more ? c + 1 : c;
    t = next ? 0 : wrap ? t + 1 : t;
    u = next ? u + 1 : u;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < k) y.p[to[i]] = gone >> i & 1 ? (T)0.0f : (T)(v[i] * d.scale);
}

// per = frame or sequence: a thread takes V columns of `runs` groups of 8 rows, loading a group at a time.  Per frame (runs is 1) a
// block decides the 8 rows of a slot and is made once for the workgroup (LDS); per sequence it decides 8 columns for as long as the
// sequence lasts, and a thread makes it again where the sequence changes: more groups a thread share the search for the first row's
// sequence and the blocks, fewer fill the card.
// LINEAR: row number times row stride is the address, padded batches included.
// Bound: HBM, read once and written once: 256 x 1024 rows of 512 float16 5.8 and 5.0 TB/s; 39 columns of bfloat16 4.0 and 3.1, two
// bytes a lane.  64 utterances of 39 floats: 5 us, the launch and the search.
template <typename T, int V, bool FRAME, bool LINEAR>
__global__ void __launch_bounds__(256) dropout_rows_kernel(const Batch b, const Split w, int runs, int64_t n_rows, const Dropout d,
                                                           const Rows<const T> x, const Rows<T> y) {
  __shared__ uint32_t rows_gone[256];
  const int slot = threadIdx.x / w.cb, group = blockIdx.y * w.cb + (threadIdx.x - slot * w.cb);
  const int64_t first = (int64_t)blockIdx.x * w.per * runs, step = (int64_t)d.at();   // the first group of 8 rows of the workgroup
  if (FRAME) {
    if (threadIdx.x < w.per) rows_gone[threadIdx.x] = philox_dropped((uint64_t)(first + threadIdx.x), step, d.seed, d.threshold);
    __syncthreads();
  }
  const int64_t r0 = (first + slot * runs) * 8;
  if (slot >= w.per || group >= w.groups || r0 >= n_rows) return;
  const int col = group * V;
  int64_t u = 0, end = n_rows;   // the sequence of a row, the first row behind it
  if (b.steps) {
    u = n_rows < ((int64_t)1 << 32) ? (int64_t)((uint32_t)r0 / (uint32_t)b.steps) : r0 / b.steps;
    end = (u + 1) * b.steps;
  } else if (!FRAME && b.off) {   // the last u with off[u] <= r0
    int64_t hi = b.n_seq;
    while (hi - u > 1) {
      const int64_t mid = (u + hi) / 2;
      if (b.off[mid] <= r0) u = mid; else hi = mid;
    }
    end = b.off[u + 1];
  }
  const int wide = (b.ncol + 7) / 8;
  auto columns = [&]() { return philox_dropped((uint64_t)u * wide + col / 8, step, d.seed, d.threshold) >> (col & 7); };
  uint32_t gone = FRAME ? 0 : columns();
  const bool split = FRAME ? !LINEAR : b.steps || b.off;
  for (int g = 0; g < runs; ++g) {
    const int64_t r = r0 + g * 8;
    const int k = (int)min((int64_t)8, n_rows - r);
    if (k <= 0) return;
    Pack<T, V> v[8];
    if (LINEAR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) load_pack<true>(v[i], x.p + (r + min(i, k - 1)) * x.rs + col);
    }
    if (FRAME) gone = rows_gone[slot];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= k) break;
      if (split && r + i >= end) {
        do end = b.steps ? end + b.steps : b.off[++u + 1]; while (r + i >= end);
        if (b.steps) u = end / b.steps - 1;
        if (!FRAME) gone = columns();
      }
      const int64_t at = LINEAR ? 0 : u * x.ss + (r + i - u * b.steps) * x.rs;
      const int64_t to = LINEAR ? (r + i) * y.rs : u * y.ss + (r + i - u * b.steps) * y.rs;
      Pack<T, V> f;
      if (LINEAR) f = v[i]; else load_pack<true>(f, x.p + at + col);
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = gone >> (FRAME ? i : j) & 1 ? 0.0f : (float)f.v[j] * d.scale;
      store_pack<true, V>(y.p + to + col, o);
    }
  }
}

}  // namespace mfcc
