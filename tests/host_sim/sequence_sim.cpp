// The operators along time built for the host, entry points, launches and kernels from their own sources: every workgroup runs
// alone, its threads as fibers that take turns at barriers, and its LDS starts as NaN, so that what a kernel reads without having
// written it shows in the result.  tests/test_sequence_kernels_cpu.py calls the entry points with host arrays.
#include <link.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <algorithm>
#include <numeric>
#include <vector>

#include "../../mfcc_amd/csrc/sequence_ops.hip"

dim3 threadIdx, blockIdx, blockDim;

namespace mfcc {
thread_local float4 shared[65536 / sizeof(float4)];   // the dynamic LDS of a launch
int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vfprintf(stderr, fmt, ap);
  fputc('\n', stderr);
  va_end(ap);
  return code;
}
}  // namespace mfcc

namespace {

constexpr size_t kStack = 64 << 10;
struct Fiber {
  ucontext_t context;
  std::vector<char> stack = std::vector<char>(kStack);
  bool done;
};
std::vector<Fiber> g_fibers(1024);
ucontext_t g_scheduler;
Fiber* g_running;
const std::function<void()>* g_body;

void entry() {
  (*g_body)();
  g_running->done = true;
  swapcontext(&g_running->context, &g_scheduler);
}

// The kernels' LDS is this module's thread-local storage.
int poison(dl_phdr_info* info, size_t, void*) {
  for (int i = 0; i < info->dlpi_phnum; ++i) {
    const auto& p = info->dlpi_phdr[i];
    if (p.p_type == PT_LOAD && (uintptr_t)&poison - (info->dlpi_addr + p.p_vaddr) < p.p_memsz) {
      for (int k = 0; k < info->dlpi_phnum; ++k)
        if (info->dlpi_phdr[k].p_type == PT_TLS) memset(info->dlpi_tls_data, 0xFF, info->dlpi_phdr[k].p_memsz);
      return 1;
    }
  }
  return 0;
}

}  // namespace

void __syncthreads() { swapcontext(&g_running->context, &g_scheduler); }

void sim_launch(dim3 grid, dim3 block, size_t shared, const std::function<void()>& thread) {
  if (shared > sizeof(mfcc::shared) || block.x > g_fibers.size()) abort();
  g_body = &thread;
  blockDim = block;
  for (unsigned y = 0; y < grid.y; ++y)
    for (unsigned x = 0; x < grid.x; ++x) {
      mfcc::shared[0].x = 0.0f;   // the storage exists from here on
      if (!dl_iterate_phdr(poison, nullptr)) abort();
      for (unsigned t = 0; t < block.x; ++t) {
        Fiber& f = g_fibers[t];
        f.done = false;
        getcontext(&f.context);
        f.context.uc_stack.ss_sp = f.stack.data();
        f.context.uc_stack.ss_size = kStack;
        f.context.uc_link = nullptr;
        makecontext(&f.context, entry, 0);
      }
      for (bool more = true, forward = true; more; forward = !forward) {   // between barriers the threads run in either order
        unsigned ended = 0;
        for (unsigned k = 0; k < block.x; ++k) {
          const unsigned t = forward ? k : block.x - 1 - k;
          if (g_fibers[t].done) {
            ++ended;
            continue;
          }
          threadIdx = dim3(t, 0, 0);
          blockIdx = dim3(x, y, 0);
          g_running = &g_fibers[t];
          swapcontext(&g_scheduler, &g_fibers[t].context);
          ended += g_fibers[t].done;
        }
        if (ended != 0 && ended != block.x) {
          fprintf(stderr, "a barrier that %u of %u threads do not reach\n", ended, block.x);
          abort();
        }
        more = ended == 0;
      }
    }
}

extern "C" mfcc_layout* sim_layout(const int64_t* counts, int64_t n) {
  auto* l = new mfcc_layout{};
  l->n_utts = n;
  l->frame_off.assign(1, 0);
  for (int64_t u = 0; u < n; ++u) l->frame_off.push_back(l->frame_off[u] + counts[u]), l->longest = std::max(l->longest, counts[u]);
  l->total_frames = l->frame_off[n];
  l->d_frame_off = l->frame_off.data();
  l->sample_off.resize(n);   // the order of falling length
  std::iota(l->sample_off.begin(), l->sample_off.end(), (int64_t)0);
  std::stable_sort(l->sample_off.begin(), l->sample_off.end(), [&](int64_t a, int64_t b) { return counts[a] > counts[b]; });
  l->d_order = l->sample_off.data();
  return l;
}
extern "C" void sim_layout_free(mfcc_layout* l) { delete l; }
// How a call divides this batch: {columns that a group has, groups of a block, groups of the last block, pieces of a sequence}
extern "C" void sim_division(int64_t n_seq, int64_t longest, int32_t ncol, int32_t* out) {
  Shape s;
  shape_of("sim_division", nullptr, n_seq, longest, ncol, 0, &s);
  const Grid g = grid_of(s);
  out[0] = g.v, out[1] = g.w.cb, out[2] = g.w.groups - (g.w.column_blocks - 1) * g.w.cb, out[3] = g.w.pieces;
}
