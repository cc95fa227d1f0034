// Operators along time over feature rows: the gated recurrence with its gradient, the running
// mean / variance normalisation and the dropout whose mask is never stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

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

constexpr int kScanTile = 8;  // rows between two checkpoints

// a = 1 / (1 + exp(-g)) and 1 - a without cancellation, from e = exp(-|g|).  The hardware exponential and reciprocal
// are good to one unit in the last place, and a product of log2(e) adds |g| 2^-24: both below the 2^-24 steps of the
// state for the gates that matter (a state with 1 - a < 1e-6 does not move).
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

// Simplest form: one thread walks one column of one sequence.
template <typename T, bool SIG>
__global__ void __launch_bounds__(256) gated_scan_kernel(const Batch b, const Rows<const T> x, const Rows<const T> g, const Rows<T> y,
                                                         const ScanPtrs q) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= b.n_seq * b.ncol) return;
  const int64_t u = i / b.ncol;
  const int c = (int)(i % b.ncol);
  const Span s = span_of(b, u);
  const T* xp = row_base(x, b, u, s) + c;
  const T* gp = row_base(g, b, u, s) + c;
  T* yp = row_base(y, b, u, s) + c;
  const int64_t dir = b.reverse ? -1 : 1;
  float h = q.h0 ? q.h0[i] : 0.0f;
  float* ck = q.ckpt ? q.ckpt + ((b.steps ? u * ((b.steps + kScanTile - 1) / kScanTile) : s.first / kScanTile + u)) * b.ncol + c : nullptr;
  for (int64_t t = 0; t < s.n; ++t) {
    if (ck && t % kScanTile == 0) ck[t / kScanTile * b.ncol] = h;
    const float xv = (float)xp[t * dir * x.rs], gv = (float)gp[t * dir * g.rs];
    float a = gv, bb = xv;
    if constexpr (SIG) {
      float na;
      sigmoid2(gv, a, na);
      bb = na * xv;
    }
    h = fmaf(a, h, bb);
    yp[t * dir * y.rs] = (T)h;
  }
  if (q.last) q.last[i] = h;
  for (int64_t t = s.n; t < b.steps; ++t) y.p[u * y.ss + t * y.rs + c] = (T)0.0f;
}

template <typename T, bool SIG>
__global__ void __launch_bounds__(256) gated_scan_backward_kernel(const Batch b, const Rows<const T> x, const Rows<const T> g,
                                                                  const Rows<const T> gy, const Rows<T> gx, const Rows<T> gg,
                                                                  const ScanPtrs q) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= b.n_seq * b.ncol) return;
  const int64_t u = i / b.ncol;
  const int c = (int)(i % b.ncol);
  const Span s = span_of(b, u);
  const T* xp = row_base(x, b, u, s) + c;
  const T* gp = row_base(g, b, u, s) + c;
  const T* yp = gy.p ? row_base(gy, b, u, s) + c : nullptr;
  T* gxp = row_base(gx, b, u, s) + c;
  T* ggp = row_base(gg, b, u, s) + c;
  const int64_t dir = b.reverse ? -1 : 1;
  float e = q.glast ? q.glast[i] : 0.0f;  // what flows into the state behind row t: a_{t+1} delta_{t+1}
  const float* ck = q.ckpt + ((b.steps ? u * ((b.steps + kScanTile - 1) / kScanTile) : s.first / kScanTile + u)) * b.ncol + c;
  for (int64_t tile = (s.n + kScanTile - 1) / kScanTile - 1; tile >= 0; --tile) {
    float hp[kScanTile], av[kScanTile], nav[kScanTile], xv[kScanTile];
    float h = ck[tile * b.ncol];
    for (int r = 0; r < kScanTile; ++r) {
      const int64_t t = tile * kScanTile + r;
      if (t < s.n) {
        xv[r] = (float)xp[t * dir * x.rs];
        av[r] = (float)gp[t * dir * g.rs];
        nav[r] = 1.0f;
        if constexpr (SIG) sigmoid2(av[r], av[r], nav[r]);
        hp[r] = h;
        h = fmaf(av[r], h, nav[r] * xv[r]);
      }
    }
    for (int r = kScanTile - 1; r >= 0; --r) {
      const int64_t t = tile * kScanTile + r;
      if (t < s.n) {
        const float d = (yp ? (float)yp[t * dir * gy.rs] : 0.0f) + e;
        gxp[t * dir * gx.rs] = (T)(nav[r] * d);
        ggp[t * dir * gg.rs] = (T)(SIG ? d * av[r] * nav[r] * (hp[r] - xv[r]) : d * hp[r]);
        e = av[r] * d;
      }
    }
  }
  if (q.gh0) q.gh0[i] = e;
  for (int64_t t = s.n; t < b.steps; ++t) {
    gx.p[u * gx.ss + t * gx.rs + c] = (T)0.0f;
    gg.p[u * gg.ss + t * gg.rs + c] = (T)0.0f;
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
