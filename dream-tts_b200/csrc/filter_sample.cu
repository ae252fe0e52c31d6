// The filtered draw of each row's next id: temperature, top-k, top-p, min-p and a given draw, per
// row, over any vocabulary (the general form of topk_sample.cu, whose order and walk it keeps).
//
//   w_j = exp((x_j - max x) / T); ids in order of value, ties by lowest id;
//   top-k keeps the first k; top-p of those the shortest prefix whose weight reaches p of theirs;
//   min-p of those the ids with w_j >= min_p; the pick is the first id at which the running
//   weight reaches u times what is left.
//
// Every filter keeps a prefix of one order, so no sort is needed: a prefix ends at a key (the
// value's order-preserving bits) and a number of the ids that share it, and each cut is found by
// a radix select over the keys that counts ids (top-k) or adds their weights (top-p, the draw).
// A weight is evaluated in 64 bits and held as an integer multiple of 2^-44: sums of up to 2^18
// of them are exact in 64 bits, so the order of the atomics cannot change a pick.
#include "tts_common.cuh"
#include "tts_internal.h"

namespace tts {

namespace {

typedef unsigned long long u64;
constexpr int kFsThreads = 512;
constexpr double kFsOne = 17592186044416.0;  // 2^44: the weight of the row's maximum

template <typename T>
TTS_DEV uint32_t fs_key(const T* x, int i) {  // 0: the id cannot be picked
  const float f = float(x[i]) + 0.f;          // -0 counts as 0
  return f > -INFINITY ? float_order_key(f) : 0u;
}
TTS_DEV float fs_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

struct FsRow {
  float mx, temp;
  // exp((x - mx) / temp); ids at the maximum weigh 1 also where it is infinite
  TTS_DEV double weight(uint32_t key) const {
    const float x = fs_value(key);
    if (x == mx) return 1.0;
    return exp((double(x) - double(mx)) / double(temp));
  }
  TTS_DEV u64 fixed(uint32_t key) const {
    return key ? u64(__double2ll_rn(weight(key) * kFsOne)) : 0ull;
  }
};

struct FsShared {
  u64 hist[256];
  u64 part[kFsThreads / 32];
  u64 value;
  uint32_t key;
  int pick;
};

// The sum of v over the CTA.
TTS_DEV u64 fs_sum(FsShared& S, u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) S.part[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = 0;
  for (int i = 0; i < kFsThreads / 32; ++i) r += S.part[i];
  return r;
}

// The first place in the order at which the running sum of f(key) over the row reaches `target`
// (>= 1, at most the whole sum): its key, and in `rest` the part of the target that the ids
// with this key have to bring.
template <typename T, typename F>
TTS_DEV uint32_t fs_select(FsShared& S, const T* x, int n, u64 target, u64* rest, F f) {
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) S.hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kFsThreads) {
      const uint32_t k = fs_key(x, i);
      if (k && (k & mask) == prefix) {
        const u64 v = f(k);
        if (v) atomicAdd(&S.hist[(k >> shift) & 255u], v);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int b = 255;
      for (; b > 0 && S.hist[b] < target; --b) target -= S.hist[b];
      S.key = prefix | (uint32_t(b) << shift);
      S.value = target;
    }
    __syncthreads();
    prefix = S.key;
    target = S.value;
    mask |= 255u << shift;
  }
  *rest = target;
  return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kFsThreads) filter_sample_kernel(const FilterSampleRequest a) {
  __shared__ FsShared S;
  const int row = blockIdx.x, t = threadIdx.x, n = a.n;
  const T* x = static_cast<const T*>(a.logits) + (size_t)row * a.ldl;
  // ---- the maximum and the first id that has it
  u64 best = 0;
  for (int i = t; i < n; i += kFsThreads) {
    const uint32_t k = fs_key(x, i);
    const u64 b = (u64(k) << 32) | uint32_t(~i);
    if (k && b > best) best = b;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 b = __shfl_xor_sync(0xffffffffu, best, o);
    best = b > best ? b : best;
  }
  if ((t & 31) == 0) S.part[t >> 5] = best;
  __syncthreads();
  for (int i = 0; i < kFsThreads / 32; ++i) best = S.part[i] > best ? S.part[i] : best;
  if (!best) {  // no id can be picked
    if (t == 0) a.out[row] = -1;
    return;
  }
  FsRow r;
  r.mx = fs_value(uint32_t(best >> 32));
  r.temp = a.temperature ? a.temperature[row] : 1.f;
  if (!(r.temp > 0.f)) {
    if (t == 0) a.out[row] = int(~uint32_t(best));
    return;
  }
  const auto weigh = [&](uint32_t k) { return r.fixed(k); };
  // ---- the weight of what each filter keeps, `left`; `cut`, the key of the last id kept (0: all are)
  u64 left = 0;
  uint32_t cut = 0;
  for (int i = t; i < n; i += kFsThreads) left += r.fixed(fs_key(x, i));
  left = fs_sum(S, left);
  const int top_k = a.top_k ? a.top_k[row] : 0;
  if (top_k > 0 && top_k < n) {
    u64 have = 0;
    for (int i = t; i < n; i += kFsThreads) have += fs_key(x, i) != 0;
    have = fs_sum(S, have);
    if (u64(top_k) < have) {
      u64 equal;
      cut = fs_select(S, x, n, u64(top_k), &equal, [](uint32_t) { return 1ull; });
      u64 above = 0;
      for (int i = t; i < n; i += kFsThreads) {
        const uint32_t k = fs_key(x, i);
        if (k > cut) above += r.fixed(k);
      }
      left = fs_sum(S, above) + equal * r.fixed(cut);
    }
  }
  const auto reach = [&](double share) {  // the running weight that `share` of `left` asks for
    const double v = ceil(share * double(left));
    return v >= double(left) ? left : v > 1. ? u64(v) : 1ull;
  };
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  if (top_p < 1.f) {
    const u64 target = reach(double(top_p));
    u64 rest;
    cut = fs_select(S, x, n, target, &rest, weigh);
    const u64 w = r.fixed(cut);
    left = target - rest + (rest + w - 1) / w * w;
  }
  const float min_p = a.min_p ? a.min_p[row] : 0.f;
  if (min_p > 0.f && (!cut || r.weight(cut) < fmin(double(min_p), 1.))) {
    u64 kept = 0;
    for (int i = t; i < n; i += kFsThreads) {
      const uint32_t k = fs_key(x, i);
      if (k && r.weight(k) >= fmin(double(min_p), 1.)) kept += r.fixed(k);
    }
    left = fs_sum(S, kept);
  }
  // ---- the draw: the key it lands on, then which of the ids that share it
  const float u = a.draws[row];
  u64 rest;
  const uint32_t key = fs_select(S, x, n, reach(u > 0.f ? double(u) : 0.), &rest, weigh);
  const u64 w = r.fixed(key);
  int skip = int((rest + w - 1) / w) - 1;  // ids with this key before the pick
  // each warp a run of ids, the runs in order
  const int per = (n + kFsThreads - 1) / kFsThreads * 32, wp = t >> 5;
  const int lo = min(n, wp * per), hi = min(n, lo + per);
  u64 mine = 0;
  for (int i = lo + (t & 31); i < hi; i += 32) mine += fs_key(x, i) == key;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if ((t & 31) == 0) S.part[wp] = mine;
  __syncthreads();
  for (int i = 0; i < wp; ++i) skip -= int(S.part[i]);
  if (skip >= 0 && skip < int(mine)) {
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + (t & 31);
      const unsigned m = __ballot_sync(0xffffffffu, i < hi && fs_key(x, i) == key);
      if (skip < __popc(m)) {
        if ((m >> (t & 31) & 1u) && __popc(m & ((1u << (t & 31)) - 1u)) == skip) a.out[row] = i;
        break;
      }
      skip -= __popc(m);
    }
  }
}

}  // namespace

cudaError_t launch_filter_sample(const FilterSampleRequest& r, cudaStream_t st) {
  if (r.f16)
    filter_sample_kernel<__half><<<r.rows, kFsThreads, 0, st>>>(r);
  else
    filter_sample_kernel<float><<<r.rows, kFsThreads, 0, st>>>(r);
  return cudaGetLastError();
}

}  // namespace tts
