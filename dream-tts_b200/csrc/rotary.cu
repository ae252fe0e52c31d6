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
// dims. The work is one read and one write of the rows: bound by HBM. A thread keeps its slot
// through several heads, so a row's table entries are read once for them, and has the heads' loads
// on their way together. (The layout is a template parameter: values indexed by a run-time choice
// of pairs went to local memory.)
//
// Measured: plain, 12345 rows of 20 f16 heads of 96 dims, tables of 131072 positions: 18.5 us (a
// copy's rate: 15.0); 77 rows of 12 f32 heads: 2.2 us. Append: about 8k rows of 32 f32 heads with
// norms 37.5 us (31.9); 4k of 36 f16 heads, interleaved, 18.8 us (11.7); 48 rows 3.3 us.
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

// A slot's 8 values as they are in memory (a thread has several heads' on their way) and as
// numbers; f16 dims that are consecutive go 16 bytes at once.
template <typename T>
struct Raw {
  uint32_t w[2 * sizeof(T)];
  TTS_DEV void load(const T* head, const Slot& s) {
    if (sizeof(T) == 4 || s.d1 == s.d0 + 4) {
      const uint4 a = *reinterpret_cast<const uint4*>(head + s.d0);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    }
    if (sizeof(T) == 4) {
      const uint4 b = *reinterpret_cast<const uint4*>(head + s.d1);
      w[sizeof(T) * 2 - 4] = b.x, w[sizeof(T) * 2 - 3] = b.y;
      w[sizeof(T) * 2 - 2] = b.z, w[sizeof(T) * 2 - 1] = b.w;
    } else if (s.d1 != s.d0 + 4) {
      const uint2 a = *reinterpret_cast<const uint2*>(head + s.d0);
      const uint2 b = *reinterpret_cast<const uint2*>(head + s.d1);
      w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
    }
  }
  TTS_DEV void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i % (2 * sizeof(T))]);
      } else if (i % 2 == 0) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i / 2]));
        v[i] = f.x, v[i + 1] = f.y;
      }
    }
  }
  static TTS_DEV void store(T* head, const Slot& s, const float* v) {
    if (sizeof(T) == 2 && s.d1 == s.d0 + 4) {
      uint4 u;
      __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<uint4*>(head + s.d0) = u;
    } else {
      Vec4<T>::store(head + s.d0, v);
      Vec4<T>::store(head + s.d1, v + 4);
    }
  }
};

// Rotates the slot's 8 values by the 4 angles from table entry 4j.
template <bool kInter>
TTS_DEV void turn(float* v, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : i + 4;
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
  int rope_len, rotary;
  int* err;
};

// Heads whose slots a thread has on their way at once. Plain rotation 4 of f16, 2 of f32 (64 bytes;
// 12345 rows of 20 f16 heads of 96: 18.5 us, one head 24.3, 8 heads 21.5).
template <typename T>
constexpr int kRotHeads = 8 / int(sizeof(T));
// The append: 8 of f16, 2 of f32, whose sum of squares and norms take more registers (about 4k
// rows of 36 f16 heads: 8 heads 18.7 us, 4 20.2, one 22.3; 8k of 32 f32 heads: 2 heads 37.5 us, 4
// 38.3, one 44.1).
template <typename T>
constexpr int kAppendHeads = sizeof(T) == 2 ? 8 : 2;

// A CTA takes `tile` rows; a thread a row's slot in kRotHeads heads, `per` = ceil(heads /
// that) heads apart (neighbouring threads read neighbouring slots and heads).
template <typename T, bool kInter>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a, int tile) {
  constexpr int kHeads = kRotHeads<T>;
  const int slots = a.hd / 8, per = (a.heads + kHeads - 1) / kHeads;
  const int items = per * slots;
  const int row0 = blockIdx.x * tile, rows = min(tile, a.rows - row0);
  for (int e = threadIdx.x; e < rows * items; e += kRotThreads) {
    const int row = row0 + e / items, in = e % items;
    const int j = in % slots, h0 = in / slots;
    const Slot s = slot_of(j, a.rotary, kInter);
    const T* src = static_cast<const T*>(a.x) + (size_t)row * a.ldx + (size_t)h0 * a.hd;
    T* dst = static_cast<T*>(a.y) + (size_t)row * a.ldy + (size_t)h0 * a.hd;
    Raw<T> x[kHeads];
#pragma unroll
    for (int u = 0; u < kHeads; ++u)
      if (h0 + u * per < a.heads) x[u].load(src + (size_t)u * per * a.hd, s);
    const int pos = a.positions[row];
    if (pos < 0 || pos >= a.rope_len) {
      if (in == 0) atomicOr(a.err, kFlagRopeRange);
      continue;
    }
    float c[4], sn[4];
    if (s.turned) {
      Vec4<float>::load(a.cos_t + (size_t)pos * (a.rotary / 2) + j * 4, c);
      Vec4<float>::load(a.sin_t + (size_t)pos * (a.rotary / 2) + j * 4, sn);
    }
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (h0 + u * per >= a.heads) break;
      float v[8];
      x[u].get(v);
      if (s.turned) turn<kInter>(v, c, sn);
      Raw<T>::store(dst + (size_t)u * per * a.hd, s, v);
    }
  }
}

// `wpr` warps a row (1, 2, 4 or 8), half a warp a head (16 slots of 8 dims, so the QK-norm's sum of
// squares is four exchanges), kAppendHeads of them at once; warps take pairs of heads in turn.
template <typename TX, typename TQ, bool kInter>
__global__ void __launch_bounds__(kRotThreads, 3) rotary_append_kernel(const RotaryAppendRequest a,
                                                                    int wpr) {
  __shared__ int starts[kChunkMaxLanes + 1];
  __shared__ alignas(16) float norms[256];
  const int t = threadIdx.x;
  if (a.norms) norms[t] = a.norms[t];
  for (int i = t; i <= a.lanes; i += kRotThreads) starts[i] = a.row_start[i];
  __syncthreads();
  if (!__syncthreads_and(chunk_starts_ok(starts, a.lanes, a.rows, t, kRotThreads))) {
    if (t == 0 && blockIdx.x == 0) atomicOr(a.err, kFlagChunkStarts);
    return;
  }
  const int wl = t & 31, j = wl & 15, half = wl >> 4;
  const int rows_at_once = kRotThreads / 32 / wpr, w = (t >> 5) % wpr;
  const int all = a.heads + 2 * a.n_kv;
  const Slot s = slot_of(j, a.rotary, kInter);
  const long cap = (long)a.max_blocks * a.block_size;
  constexpr int kHeads = kAppendHeads<TX>;
  for (int row = starts[0] + blockIdx.x * rows_at_once + (t >> 5) / wpr; row < starts[a.lanes];
       row += gridDim.x * rows_at_once) {
    const TX* src = static_cast<const TX*>(a.x) + (size_t)row * all * 128;
    Raw<TX> x[kHeads];
    const auto load = [&](int h0) {
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + 2 * wpr * u;
        if (h < all) x[u].load(src + (size_t)h * 128, s);
      }
    };
    int h0 = 2 * w + half;
    load(h0);  // on their way while the row's place is looked up
    const int lane = chunk_lane_of(starts, a.lanes, row);
    const int span = a.spans[lane];
    const int pos = span - (starts[lane + 1] - row);
    const bool outside = span < 0 || span > cap || pos >= a.rope_len;
    if (outside || pos < 0) {  // (a row before position 0 has no place: nothing is wrong with it)
      if (outside && wl == 0) atomicOr(a.err, kFlagRopeRange);
      continue;
    }
    float c[4], sn[4];
    if (s.turned) {
      Vec4<float>::load(a.cos_t + (size_t)pos * (a.rotary / 2) + j * 4, c);
      Vec4<float>::load(a.sin_t + (size_t)pos * (a.rotary / 2) + j * 4, sn);
    }
    const int page = a.block_table[(size_t)lane * a.max_blocks + pos / a.block_size];
    if (page < 0 || page >= a.num_blocks) {
      if (wl == 0) atomicOr(a.err, kFlagPageRange);
      continue;
    }
    const size_t slot = (size_t)page * a.n_kv * a.block_size + pos % a.block_size;
    for (;;) {
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int h = h0 + 2 * wpr * u;
        const bool q = h < a.heads, k = !q && h < a.heads + a.n_kv;
        float v[8];
        x[u].get(v);
        if (a.norms) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += q || k ? v[i] * v[i] : 0.f;
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          if (q || k) {
            const float r = 1.f / sqrtf(ss * (1.f / 128.f) + a.eps);
            float n[8];
            Vec4<float>::load(&norms[q ? 0 : 128] + s.d0, n);
            Vec4<float>::load(&norms[q ? 0 : 128] + s.d1, n + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * r * n[i];
          }
        }
        if (h >= all) continue;
        if ((q || k) && s.turned) turn<kInter>(v, c, sn);
        if (q) {
          Raw<TQ>::store(static_cast<TQ*>(a.q_out) + ((size_t)row * a.heads + h) * 128, s, v);
        } else {
          const int hk = h - a.heads - (k ? 0 : a.n_kv);
          Raw<__half>::store((k ? a.k_pool : a.v_pool) + (slot + (size_t)hk * a.block_size) * 128,
                             s, v);
        }
      }
      h0 += 2 * wpr * kHeads;
      if (h0 - half >= all) break;  // the same for the whole warp
      load(h0);
    }
  }
}

template <bool kInter>
void launch_append(const RotaryAppendRequest& r, int grid, int wpr, cudaStream_t st) {
  if (r.x_f16 && r.q_f16)
    rotary_append_kernel<__half, __half, kInter><<<grid, kRotThreads, 0, st>>>(r, wpr);
  else if (r.x_f16)
    rotary_append_kernel<__half, float, kInter><<<grid, kRotThreads, 0, st>>>(r, wpr);
  else if (r.q_f16)
    rotary_append_kernel<float, __half, kInter><<<grid, kRotThreads, 0, st>>>(r, wpr);
  else
    rotary_append_kernel<float, float, kInter><<<grid, kRotThreads, 0, st>>>(r, wpr);
}

}  // namespace

cudaError_t launch_rotary(const void* x, bool f16, int rows, int heads, int hd, int ldx,
                          const int* positions, const float* cos_t, const float* sin_t,
                          int rope_len, int rotary, bool interleaved, void* y, int ldy, int* err,
                          cudaStream_t st) {
  RotaryArgs a{x,   y,         rows,  heads, hd,       ldx,
               ldy, positions, cos_t, sin_t, rope_len, rotary, err};
  // rows a CTA: enough to give each thread an item, at most 8 (12345 rows of 20 f16 heads of 96: 8
  // rows 21.5 us, one row 36.6)
  const int at_once = f16 ? kRotHeads<__half> : kRotHeads<float>;
  const int items = (heads + at_once - 1) / at_once * (hd / 8);
  int tile = 1;
  while (tile < 8 && tile * items < kRotThreads) tile *= 2;
  const int grid = (rows + tile - 1) / tile;
  if (f16 && interleaved)
    rotary_kernel<__half, true><<<grid, kRotThreads, 0, st>>>(a, tile);
  else if (f16)
    rotary_kernel<__half, false><<<grid, kRotThreads, 0, st>>>(a, tile);
  else if (interleaved)
    rotary_kernel<float, true><<<grid, kRotThreads, 0, st>>>(a, tile);
  else
    rotary_kernel<float, false><<<grid, kRotThreads, 0, st>>>(a, tile);
  return cudaGetLastError();
}

cudaError_t launch_rotary_append(const RotaryAppendRequest& r, int device, cudaStream_t st) {
  // as few warps a row as still fill the SMs (8 CTAs each): rows of 32 f32 heads, 48 of them 3.3 us
  // (a warp each 8.9), about 8k 37.5 us (8 warps each 56.7)
  const int sms = num_sms(device), full = sms * 8;
  int wpr = 1;
  while (wpr < 8 && (long)r.rows * wpr < (long)full * 8) wpr *= 2;
  const int at_once = kRotThreads / 32 / wpr;
  const int need = (r.rows + at_once - 1) / at_once, grid = need < full ? need : full;
  if (r.interleaved)
    launch_append<true>(r, grid, wpr, st);
  else
    launch_append<false>(r, grid, wpr, st);
  return cudaGetLastError();
}

}  // namespace tts
