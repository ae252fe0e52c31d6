// A ragged chunk of new rows over a paged cache (tts_chunk_batch): lane i's rows are
// [row_start[i], row_start[i + 1]) and, once they are in, it holds spans[i] positions, so row j
// of its n sits at position spans[i] - n + j.
#pragma once
#include "tts_common.cuh"
#include "tts_internal.h"

namespace tts {

// Row starts that descend or leave [0, rows] make the whole batch void: a row could belong to
// two lanes. Every thread of the CTA calls this with its own part of the lanes checked.
TTS_DEV bool chunk_starts_ok(const int* starts, int lanes, int rows, int first, int step) {
  bool ok = true;
  for (int i = first; i <= lanes; i += step) {
    const int s = starts[i];
    ok = ok && s >= 0 && s <= rows && (i == lanes || s <= starts[i + 1]);
  }
  return ok;
}

// The lane that holds `row`: the largest i with starts[i] <= row, past empty lanes
// (starts[0] <= row < starts[lanes]).
TTS_DEV int chunk_lane_of(const int* starts, int lanes, int row) {
  int lo = 0, hi = lanes;  // starts[lo] <= row < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

}  // namespace tts
