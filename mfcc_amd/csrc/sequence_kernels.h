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
  int64_t n_seq;
  int64_t steps;       // 0 = packed
  int32_t ncol;
  int32_t reverse;
};

// Rows of sequence u and where its first visited row lies (sign: the direction of the visit).
struct Span {
  int64_t first, n;
};
__device__ inline Span span_of(const Batch& b, int64_t u) {
  if (!b.off) return Span{0, b.steps};
  const int64_t lo = b.off[u], n = b.off[u + 1] - lo;
  return b.steps ? Span{0, n < b.steps ? n : b.steps} : Span{lo, n};
}
template <typename T>
__device__ inline T* row_base(const Rows<T>& r, const Batch& b, int64_t u, const Span& s) {
  return r.p + (b.steps ? u * r.ss : 0) + (s.first + (b.reverse ? s.n - 1 : 0)) * r.rs;
}

// ---- the division of a batch over threads ----------------------------------------------------------
// A workgroup owns `seqs` sequences and `cb` groups of V neighbouring columns; its threads are (time slot, column group)
// pairs, `per` slots to a sequence.  A tile is per * R rows: a thread keeps the R x V values of its slot in registers,
// leaves the composition of its rows in LDS, and after one barrier composes those of the slots before it onto the state
// that enters the tile, then walks its rows from there: every value is read and written once.  A wave's load is cb * V
// neighbouring values of a row (and of the next slot's row).
constexpr int kSeqThreads = 512;
constexpr int kSlotRows = 8;   // R: composing costs per / R steps a value, registers 2 .. 6 R V

struct Split {
  int32_t groups, cb;    // column groups of a row, of a workgroup
  int32_t seqs, per;     // sequences of a workgroup, time slots of a sequence
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

// What a thread works on.  Threads behind the last slot or column group are doubles of others: they compute and write the
// same values, so that no access to rows needs a predicate as long as a tile is full.
struct Seat {
  int64_t u;           // sequence
  Span s;
  int n, sub, slot, cg, col;
  bool on;             // there is such a sequence
};
template <int V>
__device__ inline Seat seat_of(const Batch& b, const Split& w, int64_t block, int column_block) {
  Seat t;
  t.slot = threadIdx.x / w.cb;
  t.cg = min((int)threadIdx.x - t.slot * w.cb, w.groups - 1 - column_block * w.cb);
  if (t.slot >= w.seqs * w.per) t.slot = 0;
  const int g = t.slot / w.per;
  t.sub = t.slot - g * w.per;
  t.u = block * w.seqs + g;
  t.col = (column_block * w.cb + t.cg) * V;
  t.on = t.u < b.n_seq;
  t.s = t.on ? span_of(b, t.u) : Span{0, 0};
  t.n = (int)t.s.n;    // the same for all threads where a workgroup has one sequence: its tile loop runs in step
  return t;
}

// Where a thread reads the rows of its sequence from; one without rows reads the first row of the array instead (a batch
// without any rows has null arrays, and nothing is read).
template <typename T>
struct Source {
  const T* p;
  int64_t rs;
  int last;
};
template <typename T>
__device__ inline Source<T> source_of(const Rows<const T>& r, const Batch& b, const Seat& t) {
  if (t.n == 0) return Source<T>{r.p, 0, 0};
  return Source<T>{row_base(r, b, t.u, t.s) + t.col, b.reverse ? -r.rs : r.rs, t.n - 1};
}
// R rows from row t0 on.  FULL: they all exist; otherwise rows behind the end repeat the last one.  Without a branch, so
// that the loads of the next tile go out while the current one is worked on.
template <bool FULL, bool AL, typename T, int V, int R>
__device__ inline void load_rows(Pack<T, V> (&r)[R], const Source<T>& f, int t0) {
  const T* p = f.p + (FULL ? t0 : min(t0, f.last)) * f.rs;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    load_pack<AL>(r[i], p);
    p += FULL || t0 + i < f.last ? f.rs : 0;
  }
}

template <bool AL, int V, typename T>
__device__ inline void zero_behind(const Rows<T>& y, const Batch& b, const Seat& t, int per) {
  const float z[V] = {};
  for (int64_t r = t.n + t.sub; r < b.steps; r += per) store_pack<AL, V>(y.p + t.u * y.ss + r * y.rs + t.col, z);
}

// ---- gated recurrence -----------------------------------------------------------------------------
// h_t = a_t h_{t-1} + b_t is a composition of maps h -> A h + X: a run of rows is one such map, and maps of neighbouring
// runs join to (A2 A1, A2 X1 + X2).  Bound: HBM, 3 values moved a value forward and 5 backward.

// a = 1 / (1 + exp(-g)) and 1 - a without cancellation, from e = exp(-|g|).  The hardware exponential and reciprocal
// are good to one unit in the last place, and the product with log2(e) adds |g| 2^-24.
__device__ inline void sigmoid2(float g, float& a, float& na) {
  const float e = __expf(-fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  const float er = e * r;
  a = g >= 0.0f ? r : er;
  na = g >= 0.0f ? er : r;
}

struct ScanPtrs {
  const float *h0, *glast;
  float *last, *ckpt, *gh0;
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
template <bool FULL, bool AL, typename T, int V>
__device__ inline void load_tile(ScanRows<T, V>& r, const Source<T>& fx, const Source<T>& fg, int t0) {
  load_rows<FULL, AL>(r.x, fx, t0);
  load_rows<FULL, AL>(r.g, fg, t0);
}

template <typename T, int V, bool AL, bool SIG>
__global__ void __launch_bounds__(kSeqThreads, 4) gated_scan_kernel(const Batch b, const Split w, const Rows<const T> x, const Rows<const T> g,
                                                                    const Rows<T> y, const ScanPtrs q) {
  constexpr int R = kSlotRows;
  __shared__ float2 maps[2][kSeqThreads * V];
  const Seat t = seat_of<V>(b, w, blockIdx.x, blockIdx.y);
  const Source<T> fx = source_of(x, b, t), fg = source_of(g, b, t);
  const int64_t ys = b.reverse ? -y.rs : y.rs;
  T* const yp = row_base(y, b, t.u, t.s) + t.col;
  const int tile_rows = w.per * R;
  const int64_t end = t.u * b.ncol + t.col;   // of the states of a sequence
  float carry[V] = {};
  if (t.on && q.h0)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = q.h0[end + v];
  if (t.on && t.n == 0 && q.last)
#pragma unroll
    for (int v = 0; v < V; ++v) q.last[end + v] = carry[v];
  float* const ck = q.ckpt ? q.ckpt + checkpoint_row(b, t, tile_rows) * b.ncol + t.col : nullptr;

  auto work = [&](auto full, const ScanRows<T, V>& in, int tile) {
    constexpr bool FULL = full();
    const int t0 = (tile * w.per + t.sub) * R;
    const int k = FULL ? R : min(max(t.n - t0, 0), R);
    float a[R][V], x1[R][V], A[V], X[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.0f, X[v] = 0.0f;
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
    float h[V];
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
      __syncthreads();   // doubles have read their rows: y may be x
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = carry[v], carry[v] = fmaf(A[v], carry[v], X[v]);
    }
    if (FULL || k > 0) {
      if (ck && t.sub == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) ck[(int64_t)tile * b.ncol + v] = h[v];
      T* o = yp + t0 * ys;
#pragma unroll
      for (int r = 0; r < R; ++r, o += ys) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(a[r][v], h[v], x1[r][v]);
        if (FULL || r < k) store_pack<AL, V>(o, h);
      }
      if (t0 + k == t.n && q.last)
#pragma unroll
        for (int v = 0; v < V; ++v) q.last[end + v] = h[v];
    }
  };

  if (!x.p) return;
  ScanRows<T, V> in, next;
  const int full = w.seqs > 1 ? 0 : t.n / tile_rows, first = t.sub * R;
  load_tile<false, AL>(in, fx, fg, first);
  int tile = 0;
  for (; tile + 1 < full; ++tile) {
    load_tile<true, AL>(next, fx, fg, first + (tile + 1) * tile_rows);
    work(std::true_type(), in, tile);
    in = next;
  }
  if (tile < full) {
    load_tile<false, AL>(next, fx, fg, first + full * tile_rows);
    work(std::true_type(), in, tile);
    in = next;
  }
  if (w.seqs > 1 || full * tile_rows < t.n) work(std::false_type(), in, full);
  if (t.on && b.steps) zero_behind<AL, V>(y, b, t, w.per);
}

// Gradient.  With e_t = a_t delta_t, delta_t = gy_t + e_{t+1}, the way back is a composition of maps e -> A (gy + e) with the
// same products of gates, from the last tile to the first; the states h_{t-1} that dgate needs are walked
// again from the checkpoint of the tile.
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
  __shared__ float maps[2][3][kSeqThreads * V];
  const Seat t = seat_of<V>(b, w, blockIdx.x, blockIdx.y);
  const bool no_gy = !gy.p;
  const Source<T> fx = source_of(x, b, t), fg = source_of(g, b, t), fd = no_gy ? fx : source_of(gy, b, t);
  const int64_t gxs = b.reverse ? -gx.rs : gx.rs, ggs = b.reverse ? -gg.rs : gg.rs;
  T* const gxp = row_base(gx, b, t.u, t.s) + t.col;
  T* const ggp = row_base(gg, b, t.u, t.s) + t.col;
  const int tile_rows = w.per * R;
  const int64_t end = t.u * b.ncol + t.col;
  float carry[V] = {};
  if (t.on && q.glast)
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = q.glast[end + v];
  const int64_t ck_step = t.n > 0 ? b.ncol : 0;
  const float* const ck = t.n > 0 ? q.ckpt + checkpoint_row(b, t, tile_rows) * b.ncol + t.col : q.ckpt;

  auto load = [&](auto full, ScanGradRows<T, V>& r, int tile) {
    const int t0 = (tile * w.per + t.sub) * R;
    load_rows<full(), AL>(r.x, fx, t0);
    load_rows<full(), AL>(r.g, fg, t0);
    load_rows<full(), AL>(r.d, fd, t0);
    load_pack<false>(r.h, ck + tile * ck_step);
  };
  auto work = [&](auto full, const ScanGradRows<T, V>& in, int tile) {
    constexpr bool FULL = full();
    const int t0 = (tile * w.per + t.sub) * R;
    const int k = FULL ? R : min(max(t.n - t0, 0), R);
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
      T* ox = gxp + (t0 + R - 1) * gxs;
      T* og = ggp + (t0 + R - 1) * ggs;
#pragma unroll
      for (int r = R - 1; r >= 0; --r, ox -= gxs, og -= ggs) {
        float dx[V], dg[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = delta(r, v, e[v]);
          dx[v] = SIG ? na[r][v] * d : d;
          e[v] = a[r][v] * d;
          dg[v] = SIG ? e[v] * na[r][v] * (hp[r][v] - (float)in.x[r].v[v]) : d * hp[r][v];
        }
        if (FULL || r < k) {
          store_pack<AL, V>(ox, dx);
          store_pack<AL, V>(og, dg);
        }
      }
    }
  };

  ScanGradRows<T, V> in, next;
  const int full = w.seqs > 1 ? 0 : t.n / tile_rows;
  if (x.p && (w.seqs > 1 || full * tile_rows < t.n)) {
    load(std::false_type(), in, full);
    work(std::false_type(), in, full);
  }
  if (full > 0) {
    load(std::true_type(), in, full - 1);
    int tile = full - 1;
    for (; tile > 0; --tile) {
      load(std::true_type(), next, tile - 1);
      work(std::true_type(), in, tile);
      in = next;
    }
    work(std::true_type(), in, 0);
  }
  if (t.on && q.gh0 && t.sub == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) q.gh0[end + v] = carry[v];
  if (t.on && b.steps) {
    zero_behind<AL, V>(gx, b, t, w.per);
    zero_behind<AL, V>(gg, b, t, w.per);
  }
}

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

// Simplest form: one thread walks one column.  The statistics are kept in 64 bits: at a fixed point of w the roundings
// of 32 bits all have one sign (7e-6 of w off after 20000 rows at decay 0.995), and a cumulative mean of 20000 rows
// collects 20 units in the last place.
template <typename T>
__global__ void __launch_bounds__(256) running_norm_kernel(const Batch b, const Rows<const float> x, const Rows<T> y, double decay, float eps,
                                                           int center_only, const float* state_in, float* state_out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= b.n_seq * b.ncol) return;
  const int64_t u = i / b.ncol;
  const int c = (int)(i % b.ncol);
  const Span s = span_of(b, u);
  const float* xp = row_base(x, b, u, s) + c;
  T* yp = row_base(y, b, u, s) + c;
  const int64_t st = u * (1 + 2 * (int64_t)b.ncol);
  double w = 0, m = 0, q = 0;
  if (state_in) w = state_in[st], m = state_in[st + 1 + c], q = state_in[st + 1 + b.ncol + c];
  for (int64_t t = 0; t < s.n; ++t) {
    const double v = xp[t * x.rs], d = v - m;
    w = fma(decay, w, 1.0);
    const double inv = 1.0 / w;
    m = fma(d, inv, m);
    const double e = v - m;
    q = fma(decay, q, d * e);
    yp[t * y.rs] = (T)(center_only ? (float)e : (float)e * rsqrtf((float)(q * inv) + eps));
  }
  if (state_out) {
    if (c == 0) state_out[st] = (float)w;  // every column carries the same weight
    state_out[st + 1 + c] = (float)m;
    state_out[st + 1 + b.ncol + c] = (float)q;
  }
  for (int64_t t = s.n; t < b.steps; ++t) y.p[u * y.ss + t * y.rs + c] = (T)0.0f;
}

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
__device__ inline uint32_t philox_field(const uint4& w, int k) {
  const uint32_t v = (k >> 1) == 0 ? w.x : (k >> 1) == 1 ? w.y : (k >> 1) == 2 ? w.z : w.w;
  return k & 1 ? v >> 16 : v & 0xFFFFu;
}

// Simplest form: one thread per element.
template <typename T>
__global__ void __launch_bounds__(256) feature_dropout_kernel(const Batch b, int64_t n_rows, int per, uint32_t threshold, float scale,
                                                              uint64_t seed, uint64_t step, const int64_t* step_device,
                                                              const Rows<const T> x, const Rows<T> y) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n_rows * b.ncol) return;
  const int64_t r = i / b.ncol;
  const int c = (int)(i % b.ncol);
  int64_t u = 0, t = r;
  if (b.steps) {
    u = r / b.steps;
    t = r % b.steps;
  } else if (per == 2) {  // the last u with off[u] <= r
    int64_t lo = 0, hi = b.n_seq;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (b.off[mid] <= r) lo = mid; else hi = mid;
    }
    u = lo;
  }
  const uint64_t e = per == 0 ? (uint64_t)i : per == 1 ? (uint64_t)r : (uint64_t)u * ((b.ncol + 7) / 8 * 8) + c;
  const uint64_t st = step_device ? (uint64_t)*step_device : step;
  const uint32_t f = philox_field(philox4x32_10(e >> 3, st, seed), (int)(e & 7));
  const int64_t at = b.steps ? u * x.ss + t * x.rs + c : r * x.rs + c;
  const int64_t to = b.steps ? u * y.ss + t * y.rs + c : r * y.rs + c;
  y.p[to] = f < threshold ? (T)0.0f : (T)((float)x.p[at] * scale);
}

}  // namespace mfcc
