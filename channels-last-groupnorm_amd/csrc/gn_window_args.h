// Host-side interface of the attention kernels: argument block and launchers (gn_window.hip, compiled once per element type;
// the C ABI is in gn_attention.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "../../include/gnnhwc_tokens.h"
#include "gn_plan.h"

namespace gn {

constexpr int kQueries = 128;  // tokens of a workgroup's tile: 32 a wavefront

// Rows of heads: strides in bytes.
struct HeadRows {
  const void *base;
  int64_t batch_bytes, head_bytes;
  int token_bytes;
  __host__ __device__ __forceinline__ char *row(int b, int i, int h) const {
    return (char *)const_cast<void *>(base) + (int64_t)b * batch_bytes + (int64_t)i * token_bytes + (int64_t)h * head_bytes;
  }
};
enum { kInTurn = 0, kStretches = 1, kHeadsInTurn = 2 };  // which work a die takes (work_item)
struct WindowArgs {
  HeadRows q, k, v, out, dout, dq, dk, dv;
  void *rest;  // what rounding left of out, contiguous, or null
  float *lse, *delta, *largest, *part_q, *part_k, *part_v;
  const void *lengths;
  int length_type, at_end;  // at_end: the queries are the last of a sample's own tokens, not of all S
  int B, L, S, H, K, D, group;
  int left, right, sinks, causal;
  int tiles, items;           // tiles of a head, workgroups with work
  int order, per_head;        // ... of a key head
  int fine;                   // weights in twice the bits (plan_window)
  int splits;                 // out, dq: workgroups that share a row's keys
  int shares;                 // dk, dv: workgroups that share a tile's queries
  int sink_sets, sink_parts;  // dk, dv of the sinks: 32 keys each; workgroups that share the queries
  float scale, scale_log2;
  Divisor by_group, by_splits, by_tiles, by_K, by_shares, by_sink_parts, by_sink_sets, by_per_head, by_L, by_H;
  int sink_blocks;            // window_sum_kernel: workgroups that add up the sinks' parts
};

// Wavefronts of a workgroup whose wavefronts have two pairs of tiles of 32 rows each, for a head padded to `width` channels.
constexpr int window_width(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 160 ? 160 : 256; }
constexpr int few_waves(int width, int elem_size) {
  const int most = 131072 / (4 * 32 * width * elem_size);
  return most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
}

#define GN_DECLARE_WINDOW(S)                                                                  \
  hipError_t launch_window_forward_##S(const WindowArgs &a, bool few, hipStream_t stream);    \
  hipError_t launch_window_backward_##S(const WindowArgs &a, const WindowArgs &kv, const WindowArgs &sinks, hipStream_t stream);
GN_DECLARE_WINDOW(f32)
GN_DECLARE_WINDOW(f16)
GN_DECLARE_WINDOW(bf16)
#undef GN_DECLARE_WINDOW

}  // namespace gn
