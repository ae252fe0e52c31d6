// Attention of a ragged chunk of new tokens over a paged cache: row j of lane i's n new rows sits
// at position p = spans[i] - n + j and sees positions max(0, p + 1 - window) .. p of its lane
// (window 0: all of 0 .. p), grouped-query heads: o = sum_s w_s v_s / sum_s w_s,
// w_s = exp(scale q.k_s - m). A row that sees nothing (p < 0) is zero.
//
// A warp per (row, q head): 32 positions a pass, one per warp lane, the maximum and the sum
// carried from pass to pass; then the warp lanes own 4 dims each of o.
#include "chunk_batch.cuh"

namespace tts {

namespace {

constexpr int kCaThreads = 128;

template <typename TQ>
__global__ void __launch_bounds__(kCaThreads) chunk_attn_kernel(const ChunkAttnRequest a) {
  __shared__ int starts[kChunkMaxLanes + 1];
  __shared__ float qs[kCaThreads / 32][128];
  const int t = threadIdx.x, warp = t >> 5, wl = t & 31;
  for (int i = t; i <= a.lanes; i += kCaThreads) starts[i] = a.row_start[i];
  __syncthreads();
  if (!__syncthreads_and(chunk_starts_ok(starts, a.lanes, a.rows, t, kCaThreads))) {
    if (t == 0 && blockIdx.x == 0) atomicOr(a.err, kFlagChunkStarts);
    return;
  }
  const int heads = a.n_kv * a.gqa;
  const long cap = (long)a.max_blocks * a.block_size;
  const long items = (long)(starts[a.lanes] - starts[0]) * heads;
  for (long it = (long)blockIdx.x * (kCaThreads / 32) + warp; it < items;
       it += (long)gridDim.x * (kCaThreads / 32)) {
    const int row = starts[0] + int(it / heads), h = int(it % heads);
    const int lane = chunk_lane_of(starts, a.lanes, row);
    const int span = a.spans[lane];
    if (span < 0 || span > cap) {
      if (wl == 0) atomicOr(a.err, kFlagSpanRange);
      continue;
    }
    const int pos = span - (starts[lane + 1] - row);
    const int lo = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    const TQ* q = static_cast<const TQ*>(a.q) + ((size_t)row * heads + h) * 128;
    __syncwarp();
    for (int d = wl; d < 128; d += 32) qs[warp][d] = float(q[d]) * a.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = lo; s0 <= pos; s0 += 32) {
      const int s = s0 + wl;
      long at = -1;  // the position's row in the pools
      float x = -INFINITY;
      if (s <= pos) {
        const int page = a.block_table[(size_t)lane * a.max_blocks + s / a.block_size];
        if (page < 0 || page >= a.num_blocks) {
          atomicOr(a.err, kFlagPageRange);
          x = 0.f;
        } else {
          at = ((long)page * a.n_kv + h / a.gqa) * a.block_size + s % a.block_size;
          const __half2* k = reinterpret_cast<const __half2*>(a.k_pool + at * 128);
          x = 0.f;
          for (int d = 0; d < 64; ++d) {
            const float2 kk = __half22float2(k[d]);
            x += qs[warp][2 * d] * kk.x + qs[warp][2 * d + 1] * kk.y;
          }
        }
      }
      const float mn = fmaxf(m, warp_max(x));
      const float keep = m == -INFINITY ? 0.f : expf(m - mn);
      const float w = (s <= pos && mn != -INFINITY) ? expf(x - mn) : 0.f;
      l = l * keep + warp_sum(w);
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] *= keep;
      m = mn;
      const int n = min(32, pos + 1 - s0);
      for (int i = 0; i < n; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const long ai = __shfl_sync(0xffffffffu, at, i);
        if (ai < 0) continue;
        const __half2* v = reinterpret_cast<const __half2*>(a.v_pool + ai * 128 + wl * 4);
        const float2 v0 = __half22float2(v[0]), v1 = __half22float2(v[1]);
        o[0] += wi * v0.x, o[1] += wi * v0.y, o[2] += wi * v1.x, o[3] += wi * v1.y;
      }
    }
    // no visible position: zero; an l of NaN or infinity goes through to the row
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __half2* y = reinterpret_cast<__half2*>(a.out + ((size_t)row * heads + h) * 128 + wl * 4);
    y[0] = __floats2half2_rn(o[0] * inv, o[1] * inv);
    y[1] = __floats2half2_rn(o[2] * inv, o[3] * inv);
  }
}

}  // namespace

cudaError_t launch_chunk_attn(const ChunkAttnRequest& r, cudaStream_t st) {
  const long items = (long)r.rows * r.n_kv * r.gqa;
  long grid = (items + kCaThreads / 32 - 1) / (kCaThreads / 32);
  if (grid > 148L * 16) grid = 148L * 16;
  if (r.q_f16)
    chunk_attn_kernel<__half><<<int(grid), kCaThreads, 0, st>>>(r);
  else
    chunk_attn_kernel<float><<<int(grid), kCaThreads, 0, st>>>(r);
  return cudaGetLastError();
}

}  // namespace tts
