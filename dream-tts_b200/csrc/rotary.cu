// Rotary positions beyond the decode step's fixed form: half-split or interleaved pairs, the
// first rotary_dim dims of each head, caller-made tables (scaled ones for long contexts), over
// plain rows at per-row positions and over a ragged chunk whose K and V rows go into a paged
// cache (with the optional QK-norm of crates/tts-nn/src/qkrope.rs:26-69 before the rotation).
//
// Pair (a, b) at angle t becomes (a cos t - b sin t, b cos t + a sin t): dims (i, i + r/2) in the
// half layout, (2i, 2i + 1) interleaved, r = rotary_dim; dims past r pass through.
//
// A head is cut into slots of 8 dims that one thread loads, turns and stores, holding whole
// pairs: in the half layout slot j < r/8 is dims 4j..4j+3 and r/2 + 4j..+3, else 8 consecutive
// dims. The work is one read and one write of the rows; the table rows are shared by the heads.
#include "chunk_batch.cuh"

namespace tts {

namespace {

constexpr int kRotThreads = 256;

template <typename T>
struct Vec4;
template <>
struct Vec4<float> {
  static TTS_DEV void load(const float* p, float* v) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  }
  static TTS_DEV void store(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Vec4<__half> {
  static TTS_DEV void load(const __half* p, float* v) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
  static TTS_DEV void store(__half* p, const float* v) {
    uint2 u;
    *reinterpret_cast<__half2*>(&u.x) = __floats2half2_rn(v[0], v[1]);
    *reinterpret_cast<__half2*>(&u.y) = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = u;
  }
};

// The two runs of 4 dims that slot j of a head holds.
struct Slot {
  int d0, d1;
  bool turned;
};
TTS_DEV Slot slot_of(int j, int rotary, int interleaved) {
  Slot s;
  s.turned = j * 8 < rotary;
  if (s.turned && !interleaved) {
    s.d0 = j * 4;
    s.d1 = rotary / 2 + j * 4;
  } else {
    s.d0 = j * 8;
    s.d1 = j * 8 + 4;
  }
  return s;
}

// Rotates the slot's 8 values by the 4 angles from table entry 4j.
TTS_DEV void turn(float* v, const float* c, const float* s, int interleaved) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : i + 4;
    const float a = v[ia], b = v[ib];
    v[ia] = a * c[i] - b * s[i];
    v[ib] = b * c[i] + a * s[i];
  }
}

struct RotaryArgs {
  const void* x;
  void* y;
  int rows, heads, hd, ldx, ldy;
  const int* positions;
  const float* cos_t;
  const float* sin_t;
  int rope_len, rotary, interleaved;
  int* err;
};

// A thread per (row, head, slot).
template <typename T>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  const int slots = a.hd / 8;
  const long total = (long)a.rows * a.heads * slots;
  for (long e = blockIdx.x * (long)kRotThreads + threadIdx.x; e < total;
       e += (long)gridDim.x * kRotThreads) {
    const int j = int(e % slots);
    const long rh = e / slots;
    const int h = int(rh % a.heads), row = int(rh / a.heads);
    const int pos = a.positions[row];
    if (pos < 0 || pos >= a.rope_len) {
      if (h == 0 && j == 0) atomicOr(a.err, kFlagRopeRange);
      continue;
    }
    const Slot s = slot_of(j, a.rotary, a.interleaved);
    const T* src = static_cast<const T*>(a.x) + (size_t)row * a.ldx + (size_t)h * a.hd;
    T* dst = static_cast<T*>(a.y) + (size_t)row * a.ldy + (size_t)h * a.hd;
    float v[8];
    Vec4<T>::load(src + s.d0, v);
    Vec4<T>::load(src + s.d1, v + 4);
    if (s.turned) {
      float c[4], sn[4];
      Vec4<float>::load(a.cos_t + (size_t)pos * (a.rotary / 2) + j * 4, c);
      Vec4<float>::load(a.sin_t + (size_t)pos * (a.rotary / 2) + j * 4, sn);
      turn(v, c, sn, a.interleaved);
    }
    Vec4<T>::store(dst + s.d0, v);
    Vec4<T>::store(dst + s.d1, v + 4);
  }
}

// One CTA per run of rows; half a warp per head of a row (16 slots of 8 dims), so the QK-norm's
// sum of squares is four exchanges.
template <typename TX, typename TQ>
__global__ void __launch_bounds__(kRotThreads) rotary_append_kernel(const RotaryAppendRequest a) {
  __shared__ int starts[kChunkMaxLanes + 1];
  const int t = threadIdx.x;
  for (int i = t; i <= a.lanes; i += kRotThreads) starts[i] = a.row_start[i];
  __syncthreads();
  if (!__syncthreads_and(chunk_starts_ok(starts, a.lanes, a.rows, t, kRotThreads))) {
    if (t == 0 && blockIdx.x == 0) atomicOr(a.err, kFlagChunkStarts);
    return;
  }
  const int j = t & 15, group = t >> 4;
  const int all = a.heads + 2 * a.n_kv;
  const Slot s = slot_of(j, a.rotary, a.interleaved);
  const long cap = (long)a.max_blocks * a.block_size;
  for (int row = starts[0] + blockIdx.x; row < starts[a.lanes]; row += gridDim.x) {
    const int lane = chunk_lane_of(starts, a.lanes, row);
    const int span = a.spans[lane];
    const int pos = span - (starts[lane + 1] - row);
    if (span > cap || pos < 0 || pos >= a.rope_len) {
      if (t == 0) atomicOr(a.err, kFlagRopeRange);
      continue;
    }
    const int page = a.block_table[(size_t)lane * a.max_blocks + pos / a.block_size];
    if (page < 0 || page >= a.num_blocks) {
      if (t == 0) atomicOr(a.err, kFlagPageRange);
      continue;
    }
    float c[4], sn[4];
    if (s.turned) {
      Vec4<float>::load(a.cos_t + (size_t)pos * (a.rotary / 2) + j * 4, c);
      Vec4<float>::load(a.sin_t + (size_t)pos * (a.rotary / 2) + j * 4, sn);
    }
    const size_t slot = (size_t)page * a.n_kv * a.block_size + pos % a.block_size;
    for (int h0 = 0; h0 < all; h0 += kRotThreads / 16) {
      const int h = h0 + group;
      const bool live = h < all;
      float v[8];
      if (live) {
        const TX* src = static_cast<const TX*>(a.x) + ((size_t)row * all + h) * 128;
        Vec4<TX>::load(src + s.d0, v);
        Vec4<TX>::load(src + s.d1, v + 4);
      }
      const bool qk = live && h < a.heads + a.n_kv;
      if (a.norms) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += qk ? v[i] * v[i] : 0.f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (qk) {
          const float r = 1.f / sqrtf(ss * (1.f / 128.f) + a.eps);
          const float* w = a.norms + (h < a.heads ? 0 : 128);
          float w8[8];
          Vec4<float>::load(w + s.d0, w8);
          Vec4<float>::load(w + s.d1, w8 + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w8[i];
        }
      }
      if (!live) continue;
      if (qk && s.turned) turn(v, c, sn, a.interleaved);
      if (h < a.heads) {
        TQ* dst = static_cast<TQ*>(a.q_out) + ((size_t)row * a.heads + h) * 128;
        Vec4<TQ>::store(dst + s.d0, v);
        Vec4<TQ>::store(dst + s.d1, v + 4);
      } else {
        const int hk = h - a.heads;
        __half* pool = hk < a.n_kv ? a.k_pool : a.v_pool;
        __half* dst = pool + (slot + (size_t)(hk % a.n_kv) * a.block_size) * 128;
        Vec4<__half>::store(dst + s.d0, v);
        Vec4<__half>::store(dst + s.d1, v + 4);
      }
    }
  }
}

int grid_for(long items, long per) {
  const long g = (items + per - 1) / per;
  return int(g < 1 ? 1 : g > 148L * 32 ? 148L * 32 : g);
}

}  // namespace

cudaError_t launch_rotary(const void* x, bool f16, int rows, int heads, int hd, int ldx,
                          const int* positions, const float* cos_t, const float* sin_t,
                          int rope_len, int rotary, bool interleaved, void* y, int ldy, int* err,
                          cudaStream_t st) {
  RotaryArgs a{x,     y,     rows,     heads,  hd,          ldx, ldy, positions,
               cos_t, sin_t, rope_len, rotary, interleaved, err};
  const int grid = grid_for((long)rows * heads * (hd / 8), kRotThreads);
  if (f16)
    rotary_kernel<__half><<<grid, kRotThreads, 0, st>>>(a);
  else
    rotary_kernel<float><<<grid, kRotThreads, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_rotary_append(const RotaryAppendRequest& r, cudaStream_t st) {
  const int grid = grid_for(r.rows, 1);
  if (r.x_f16 && r.q_f16)
    rotary_append_kernel<__half, __half><<<grid, kRotThreads, 0, st>>>(r);
  else if (r.x_f16)
    rotary_append_kernel<__half, float><<<grid, kRotThreads, 0, st>>>(r);
  else if (r.q_f16)
    rotary_append_kernel<float, __half><<<grid, kRotThreads, 0, st>>>(r);
  else
    rotary_append_kernel<float, float><<<grid, kRotThreads, 0, st>>>(r);
  return cudaGetLastError();
}

}  // namespace tts
