// The handle behind pf_handle: per-device state shared by the entry points of
// the library's translation units.
#pragma once

#include "pf_common.cuh"

// The selector's decision for one matrix.
struct pf_variant_choice {
  int variant;  // a PF_VARIANT_* other than AUTO
  int lanes;    // lanes per row for the row-group variants (ROWVEC, ROWGROUP)
};

struct pf_select_entry {
  const void *row_ptr;
  int64_t m, nnz;
  int idx_bytes;
  pf_variant_choice choice;
};

// Per-device state: the selector cache, scratch for cut-row carries and the
// long-row chunks, the fused step's norm partials, the device error word, and
// the buffers of the host-buffer entry points.
struct pf_handle_s {
  int device = 0;
  int num_sms = 0;
  int variant = PF_VARIANT_AUTO;
  // selector cache: decision per (row_ptr, m, nnz); any variant is correct
  // for any matrix, so a stale entry can only cost speed
  pf_select_entry cache[16];
  int cache_n = 0, cache_next = 0;
  int64_t *sample_dev = nullptr;
  int64_t *sample_host = nullptr;  // pinned
  int64_t slice_override = 0;  // testing knob: fixed nnz per slice (NNZSPLIT, NNZROW)
  // cut-row scratch
  double *carry = nullptr;     // 2 * cap doubles (head, tail)
  unsigned *counters = nullptr;
  int64_t cap = 0;
  bool scratch_dirty = false;
  unsigned *err = nullptr;
  // fused all-gather: per-CTA norm partials + counter (zeroed when grown)
  double *dist_part = nullptr;
  unsigned *dist_counter = nullptr;
  unsigned long long *dist_wait = nullptr;  // step-barrier wait, ns summed over CTAs
  int64_t dist_grid = 0;                    // CTAs of the last fused launch
  int64_t dist_cap = 0;
  // grouped products with split sums: the parts' sums (128 x 128 for each SM) and,
  // behind them, four counters for each SM (all zero between calls). One
  // allocation, never replaced.
  float *gmm_partial = nullptr;
  unsigned *gmm_arrived = nullptr;
  size_t gmm_counters() const { return (size_t)num_sms * 4; }
  // host-call buffers, and the copy stream and events of the pipelined
  // host call (created on first use)
  void *hbuf[5] = {nullptr, nullptr, nullptr, nullptr, nullptr};
  size_t hcap[5] = {0, 0, 0, 0, 0};
  cudaStream_t hcopy = nullptr;
  cudaEvent_t hev[17] = {};
};
