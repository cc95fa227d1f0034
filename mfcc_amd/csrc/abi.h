// Host-side pieces that the translation units of the library share: the error text of the calling
// thread, the check of a HIP call, the launch-size helper and the batch layout.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

#include "../../include/mfcc_amd.h"

namespace mfcc {
struct Tile;
// Stores the text for mfcc_last_error() and returns `code`.
__attribute__((visibility("hidden"))) int fail(int code, const char* fmt, ...);
}  // namespace mfcc

#define HIP_TRY(expr)                                                                              \
  do {                                                                                             \
    hipError_t e_ = (expr);                                                                        \
    if (e_ != hipSuccess) return mfcc::fail(MFCC_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

inline unsigned blocks_for(int64_t n, int per) { return (unsigned)((n + per - 1) / per); }

struct mfcc_layout {
  int device;
  int64_t n_utts, total_samples, total_frames;
  int64_t longest = 0;  // most frames in one utterance
  std::vector<int64_t> sample_off, frame_off;
  int64_t* d_sample_off = nullptr;
  int64_t* d_frame_off = nullptr;
  int64_t* d_order = nullptr;  // utterances by falling frame count, behind the offsets in the same allocation; frames_only layouts of unequal counts
  mfcc::Tile* d_tiles = nullptr;
  int64_t n_tiles;
  // the same frames cut for the persistent workgroups of split_kernel.h: workgroup w walks
  // d_wg_tiles[d_wg_off[w] .. d_wg_off[w + 1]); every workgroup gets about the same number of batches
  mfcc::Tile* d_wg_tiles = nullptr;
  int32_t* d_wg_off = nullptr;
  int32_t n_wg = 0;
  bool frames_only = false;  // made by mfcc_layout_create_frames: frame offsets only, no audio geometry
  // what the tile list was cut for: a plan may only run on a layout of its own framing whose
  // tiles fit its kernel
  int32_t frame_size = 0, frame_step = 0, frame_rule = 0;
  int32_t max_nt = 0;  // most output frames in one tile
  bool general_cut = false;  // tiles cut for the general kernel (no halo rule)
};
