// The filtered draw of each row's next id: temperature, top-k, top-p, min-p and a given draw, per
// row, over any vocabulary (the general form of topk_sample.cu, whose order and walk it keeps).
//
//   w_j = exp((x_j - max x) / T); ids in order of value, ties by lowest id;
//   top-k keeps the first k; top-p of those the shortest prefix whose weight reaches p of theirs;
//   min-p of those the ids with w_j >= min_p; the pick is the first id at which the running
//   weight reaches u times what is left.
//
// Every filter keeps a prefix of one order, so no sort of the row is needed. A cluster of CTAs
// holds the row in shared memory (it is read from HBM once), finds the maximum, and adds up counts
// and weights in 1024 bins of equal width in log w. A cut or the draw then falls into one bin,
// found by a scan; only that bin's ids are gathered into the first CTA, sorted and walked. Where
// the first filter leaves few ids, all of them are gathered at once and the rest happens there.
// A bin with too many ids (equal logits) is narrowed by the bits of its keys. Counts are kept only
// where top-k asks for them.
//
// A weight is evaluated in 64 bits and held as an integer multiple of 2^-44 of the largest: sums of
// up to 2^18 of them are exact in 64 bits, so neither the order of the atomics nor the number of
// CTAs can change a pick. The rounding can move a border between two ids by 2^-45 for each id before
// it, so a draw or cut that near to one may take its neighbour (seen with draws of 1 - 2^-24 over 75
// thousand ids and more, where ids weigh about 1e-11; for draws at large the chance is below 1e-7).
//
// Measured (192 rows of 151851 f32 ids, top-p 0.9): 233 us; reading them once takes 18. What bounds
// it is the chain of a row's steps (load, maximum, bins, exchange, cut, draw), each behind a
// barrier of the CTA or cluster: issue slots are 41 % used, a row alone takes 30 us, and some 36
// rows are at work at a time. So the row stays in shared memory, two CTAs share an SM, and CTAs
// exchange little. (The bins cost 61 us of it in atomics, 32 bits at a time: 64 at once, 319 us;
// of 247 us then, 512 bins took 276, 2048 took 247, clusters of 16 CTAs 399 to 461.) 48 rows of
// 32003 with every filter 22 us, 8 rows of 2048 with top-k alone 10 us.
#include <cfloat>
#include <mutex>

#include "tts_common.cuh"
#include "tts_internal.h"

namespace tts {

namespace {

typedef unsigned long long u64;
constexpr int kFsThreads = 512;
constexpr int kFsWarps = kFsThreads / 32;
constexpr int kFsBins = 1024;
constexpr int kFsLoads = 4;      // 16-byte loads a thread has on their way
constexpr int kFsCap = 1024;     // ids the first CTA sorts at once
// ... without cutting the list into parts first (512 rows of 32000: 121 us, 125 where only 96 are;
// 192 rows of 151851, lists of 600: 247 us, 287 where all are)
constexpr int kFsFew = 256;
constexpr int kFsMaxCluster = 8;
constexpr float kFsOctaves = 45.f;  // below 2^-45 a weight is 0
// Ids in a CTA's part up to which two CTAs share an SM (192 rows of 151851: two 247 us, one with
// twice the part 256; 512 rows of 32000: 129 and 136).
constexpr int kFsTwo = 19456;
constexpr double kFsOne = 17592186044416.0;  // 2^44: the weight of the row's maximum

// Counts and 64-bit weights, the latter in two words each.
template <int N>
struct FsSums {
  uint32_t count[N], lo[N], hi[N];
  __device__ __forceinline__ u64 weight(int i) const { return (u64(hi[i]) << 32) + lo[i]; }
  __device__ __forceinline__ void put(int i, u64 w, uint32_t c) {
    lo[i] = uint32_t(w), hi[i] = uint32_t(w >> 32), count[i] = c;
  }
  // One id more: the carry of the lower word goes up.
  __device__ __forceinline__ void add(int i, u64 w, bool with_count) {
    if (with_count) atomicAdd(&count[i], 1u);
    if (!w) return;
    const uint32_t low = uint32_t(w), old = atomicAdd(&lo[i], low);
    const uint32_t up = uint32_t(w >> 32) + (old + low < old ? 1u : 0u);
    if (up) atomicAdd(&hi[i], up);
  }
};

struct FsSmem {
  FsSums<kFsBins> bin;          // by bin, then running
  FsSums<256> digit;            // by 8 bits of the keys, in a bin too full to sort
  alignas(16) u64 list[kFsCap];  // first CTA: gathered ids, key << 32 | ~id
  u64 run[kFsCap];              // their running weights (before: this CTA's gathered ids)
  double exp_table[256];        // 2^(i / 256)
  u64 part[kFsWarps];
  float low[kFsWarps];
  uint32_t floor[kFsMaxCluster];  // by CTA: its smallest value's bits
  u64 share[2][kFsMaxCluster];  // one value of each CTA, two uses in turn
  u64 answer;                   // what one thread, or the first CTA, found
  uint32_t mine;                // ids this CTA gathers
  int found;                    // by fs_reach
  int digit_at;                 // the part of the keys that a target falls into
  u64 digit_below[2];           // and the weight and count above it
  alignas(16) float x[4];       // this CTA's part of the row (a.per entries), -inf: never picked
};

// NaN is not to be picked, -0 is 0.
TTS_DEV float fs_clean(float f) { return f > -INFINITY ? f + 0.f : -INFINITY; }
TTS_DEV float fs_value(uint32_t key) {  // of float_order_key
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// ---- shared memory of the cluster's CTAs
TTS_DEV uint32_t ld_cluster(const uint32_t* p, uint32_t cta) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, cta)) : "memory");
  return v;
}
TTS_DEV void st_cluster(uint32_t* p, uint32_t cta, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(p, cta)), "r"(v) : "memory");
}
TTS_DEV void st_cluster(u64* p, uint32_t cta, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_addr(p, cta)), "l"(v) : "memory");
}
TTS_DEV uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// A row's scale. 2^t = 2^(i / 256) 2^r with i the integer nearest 256 t: the first factor from a
// table (and the exponent), the second by its Taylor series (|r| <= 2^-9, the first term left out
// below 2^-54 of the sum).
struct FsScale {
  float mx, per_bin;  // the row's maximum; bins per unit of x
  double c;           // log2(e) / T
  const double* table;
  // Grows as x falls (0 for the maximum, also where the scale is infinite and this is 0 times it).
  TTS_DEV int bin(float x) const { return min(kFsBins - 1, int((mx - x) * per_bin)); }
  // Values below and above all of the given bins', one bin wider than they are.
  TTS_DEV void bounds(int bin0, int bin1, float* low, float* high) const {
    *low = bin1 == kFsBins - 1 ? -INFINITY : mx - (bin1 + 2) / per_bin;
    *high = bin0 < 2 ? INFINITY : mx - (bin0 - 1) / per_bin;
  }
  TTS_DEV u64 weight(float x) const {
    const double t = (double(x) - double(mx)) * c;
    const double magic = 26388279066624.;  // 1.5 * 2^44: one unit of the sum's last place is 2^-8
    const double s = t + magic;
    const int i = __double2loint(s);
    const double r = t - (s - magic);
    double p = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);  // ln 2^n / n!
    p = fma(p, r, 2.402265069591007e-1);
    p = fma(p, r, 6.931471805599453e-1);
    p = fma(p, r, 1.);
    const double v = p * table[i & 255];
    // times 2^(44 + i / 256) by the exponent, then rounded to an integer by the last place of 2^52
    const double f = __hiloint2double(__double2hiint(v) + ((44 + (i >> 8)) << 20),
                                      __double2loint(v));
    const u64 w = u64(__double_as_longlong(f + 4503599627370496.)) & 0xfffffffffffffull;
    return t > -double(kFsOctaves) ? w : 0;  // no branch: the steps above are harmless for any t
  }
};

// The sum of v over the CTA, in every thread.
TTS_DEV u64 fs_sum(FsSmem& S, u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) S.part[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = 0;
#pragma unroll
  for (int i = 0; i < kFsWarps; ++i) r += S.part[i];
  return r;
}
// The sum of v over the threads before this one.
TTS_DEV u64 fs_before(FsSmem& S, u64 v) {
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
    if ((threadIdx.x & 31) >= o) inc += x;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 31) S.part[threadIdx.x >> 5] = inc;
  __syncthreads();
  u64 r = inc - v;
#pragma unroll
  for (int i = 0; i < kFsWarps - 1; ++i) r += i < int(threadIdx.x >> 5) ? S.part[i] : 0;
  return r;
}

// The first place at which a running sum (inclusive, `n` entries) reaches `target`: `n` if none.
template <typename F>
TTS_DEV int fs_reach(FsSmem& S, int n, u64 target, F sum_at) {
  __syncthreads();
  if (threadIdx.x == 0) S.found = n;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kFsThreads)
    if (sum_at(i) >= target && (i == 0 || sum_at(i - 1) < target)) S.found = i;
  __syncthreads();
  return S.found;
}

// The sums of the row's CTAs, in all of them: each adds up a share of the entries.
template <int N>
TTS_DEV void fs_join(FsSums<N>& s, uint32_t rank, uint32_t ctas) {
  cluster_sync();
  if (ctas == 1) return;
  const int share = (N + int(ctas) - 1) / int(ctas), b0 = int(rank) * share;
  for (int e = threadIdx.x; e < 2 * share; e += kFsThreads) {
    const int b = b0 + (e >> 1);  // an entry's count and its weight by a thread each
    if (b >= N) continue;
    uint32_t l[kFsMaxCluster], h[kFsMaxCluster];
#pragma unroll
    for (uint32_t i = 0; i < kFsMaxCluster; ++i) {
      l[i] = i < ctas ? ld_cluster(e & 1 ? &s.lo[b] : &s.count[b], i) : 0;
      h[i] = i < ctas && (e & 1) ? ld_cluster(&s.hi[b], i) : 0;
    }
    u64 w = 0;
#pragma unroll
    for (uint32_t i = 0; i < kFsMaxCluster; ++i) w += (u64(h[i]) << 32) + l[i];
    for (uint32_t i = 0; i < ctas; ++i) {  // only this thread reads or writes these words
      st_cluster(e & 1 ? &s.lo[b] : &s.count[b], i, uint32_t(w));
      if (e & 1) st_cluster(&s.hi[b], i, uint32_t(w >> 32));
    }
  }
  cluster_sync();
}

// Every CTA's v (alike in its threads) in all of the row's CTAs. One cluster barrier: the array is
// used two uses later at the earliest, when all have passed the next use's barrier and so have
// read this one.
struct FsShare {
  int turn = 0;
  TTS_DEV const u64* operator()(FsSmem& S, u64 v, uint32_t rank, uint32_t ctas) {
    u64* at = S.share[turn];
    turn ^= 1;
    if (threadIdx.x < ctas) st_cluster(&at[rank], threadIdx.x, v);
    cluster_sync();
    return at;
  }
};

// f(i, x) for this CTA's `n` values that may be picked, four to a load.
template <typename F>
TTS_DEV void fs_each(const FsSmem& S, int n, F f) {
  for (int i = threadIdx.x * 4; i < n; i += kFsThreads * 4) {
    const float4 v = *reinterpret_cast<const float4*>(S.x + i);  // padded to fours with -inf
    if (v.x > -INFINITY) f(i, v.x);
    if (v.y > -INFINITY) f(i + 1, v.y);
    if (v.z > -INFINITY) f(i + 2, v.z);
    if (v.w > -INFINITY) f(i + 3, v.w);
  }
}

// f(i, x) for those of them from low to high (both finite or low below all), where they are few.
template <typename F>
TTS_DEV void fs_each_in(const FsSmem& S, int n, float low, float high, F f) {
  low = fmaxf(low, -FLT_MAX);  // not the padding, nor what may not be picked
#pragma unroll 2
  for (int i = threadIdx.x * 4; i < n; i += kFsThreads * 4) {
    const float4 v = *reinterpret_cast<const float4*>(S.x + i);
    const bool x = v.x >= low && v.x <= high, y = v.y >= low && v.y <= high,
               z = v.z >= low && v.z <= high, w = v.w >= low && v.w <= high;
    if (!(x || y || z || w)) continue;
    if (x) f(i, v.x);
    if (y) f(i + 1, v.y);
    if (z) f(i + 2, v.z);
    if (w) f(i + 3, v.w);
  }
}

// Counts the row's ids of the given bins and keys and, if the first CTA's list holds them all, puts
// them there, each CTA's behind those of the CTAs before it.
TTS_DEV int fs_gather(FsSmem& S, const FsScale& r, int n, int id0, uint32_t rank, uint32_t ctas,
                      FsShare& share, int bin0, int bin1, uint32_t key0, uint32_t key1) {
  const int t = threadIdx.x;
  float low, high;
  r.bounds(bin0, bin1, &low, &high);
  __syncthreads();
  if (t == 0) S.mine = 0;
  __syncthreads();
  fs_each_in(S, n, low, high, [&](int i, float x) {
    const int b = r.bin(x);
    const uint32_t k = float_order_key(x);
    if (b < bin0 || b > bin1 || k < key0 || k > key1) return;
    const uint32_t at = atomicAdd(&S.mine, 1u);
    if (at < uint32_t(kFsCap)) S.run[at] = (u64(k) << 32) | uint32_t(~(id0 + i));
  });
  __syncthreads();
  const int m = int(S.mine);
  const u64* of = share(S, u64(m), rank, ctas);
  int all = 0, place = 0;
  for (uint32_t i = 0; i < ctas; ++i) {
    if (i == rank) place = all;
    all += int(of[i]);
  }
  if (all <= kFsCap) {
    for (int i = t; i < m; i += kFsThreads) st_cluster(&S.list[place + i], 0, S.run[i]);
    cluster_sync();
  }
  return all;
}
// First CTA: sorts the list's m entries by key, then id, and runs their weights up.
TTS_DEV void fs_sort(FsSmem& S, const FsScale& r, int m) {
  const int t = threadIdx.x;
  // Each entry's place is the number of larger ones: warps of 32 entries, and where those are few
  // several warps to the same 32, each counting over a part of the list.
  const int groups = (m + 31) / 32, parts = max(1, kFsWarps / groups);
  const int each = (m + parts - 1) / parts;
  const int pad = (m + 1) / 2 * 2;
  if (t == 0 && pad > m) S.list[m] = 0;
  int* place = reinterpret_cast<int*>(S.run);  // not in use now
  for (int i = t; i < m; i += kFsThreads) place[i] = 0;
  __syncthreads();
  u64 e[2] = {0, 0};
  int at[2] = {-1, -1};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int wp = (t >> 5) + u * kFsWarps;
    const int g = wp % groups, part = wp / groups;
    if (part >= parts || (u == 1 && groups <= kFsWarps)) continue;
    const int i = g * 32 + (t & 31);
    if (part == 0 && i < m) e[u] = S.list[i], at[u] = i;
    const u64 mine = i < m ? S.list[i] : ~0ull;
    int larger = 0;
    const int from = part * each & ~1;
    const int to = part == parts - 1 ? pad : min(pad, (part + 1) * each & ~1);
#pragma unroll 4
    for (int j = from; j < to; j += 2) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&S.list[j]);
      larger += (x.x > mine) + (x.y > mine);
    }
    if (i < m && larger) atomicAdd(&place[i], larger);
  }
  __syncthreads();
  int to[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) to[u] = at[u] >= 0 ? place[at[u]] : 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (at[u] >= 0) S.list[to[u]] = e[u];
  __syncthreads();
  constexpr int kPer = kFsCap / kFsThreads;
  u64 w[kPer], sum = 0;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int i = t * kPer + u;
    w[u] = i < m ? r.weight(fs_value(uint32_t(S.list[i] >> 32))) : 0;
    sum += w[u];
  }
  sum = fs_before(S, sum);
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    sum += w[u];
    S.run[t * kPer + u] = sum;
  }
  __syncthreads();
}

// Which of the 256 parts the running count (`ids`) or weight reaches `rest` in, from the largest
// keys down; `rest` and `below` move to that part's start. Returns the part.
TTS_DEV int fs_part(FsSmem& S, bool ids, u64* rest, u64* below) {
  const int t = threadIdx.x, part = 255 - t;
  const u64 w = t < 256 ? S.digit.weight(part) : 0, c = t < 256 ? S.digit.count[part] : 0;
  const u64 w0 = fs_before(S, w), c0 = fs_before(S, c);
  const u64 step = ids ? c : w, step0 = ids ? c0 : w0;
  if (t < 256 && step0 < *rest && *rest <= step0 + step) {
    S.digit_at = part;
    S.digit_below[0] = w0;
    S.digit_below[1] = c0;
  }
  __syncthreads();
  *below += S.digit_below[0];
  *rest -= S.digit_below[ids ? 1 : 0];
  return S.digit_at;
}

// Where the running count (`ids`) or weight of the order reaches `target` (at least 1, at most
// all): the weight up to there, the id there included. With `out` that id goes there. All of the
// row's CTAs call it.
TTS_DEV u64 fs_resolve(FsSmem& S, const FsScale& r, int n, int id0, uint32_t rank, uint32_t ctas,
                       FsShare& share, bool ids, u64 target, int* out) {
  const int t = threadIdx.x;
  const int bin = fs_reach(S, kFsBins, target, [&](int i) {
    return ids ? u64(S.bin.count[i]) : S.bin.weight(i);
  });
  u64 below = bin ? S.bin.weight(bin - 1) : 0;  // the weight of the ids before those looked at
  u64 rest = target - (ids ? (bin ? u64(S.bin.count[bin - 1]) : 0) : below);
  uint32_t key0 = 1, key1 = 0xffffffffu;
  int members = fs_gather(S, r, n, id0, rank, ctas, share, bin, bin, key0, key1);
  {
    float low, high;
    r.bounds(bin, bin, &low, &high);
    key0 = max(float_order_key(low), 1u), key1 = float_order_key(high);
  }
  while (members > kFsCap && key0 < key1) {
    // 256 equal parts of the keys, then the one that the target falls into
    const int shift = max(0, 24 - __clz(key1 - key0));
    __syncthreads();
    if (t < 256) S.digit.put(t, 0, 0);
    __syncthreads();
    fs_each(S, n, [&](int, float x) {
      const uint32_t k = float_order_key(x);
      if (k >= key0 && k <= key1 && r.bin(x) == bin)
        S.digit.add((k - key0) >> shift, r.weight(x), true);
    });
    fs_join(S.digit, rank, ctas);
    const int d = fs_part(S, ids, &rest, &below);
    members = int(S.digit.count[d]);
    key0 += uint32_t(d) << shift;
    key1 = key0 + min(key1 - key0, (1u << shift) - 1u);
    cluster_sync();  // all CTAs have read the sums
    if (members <= kFsCap) fs_gather(S, r, n, id0, rank, ctas, share, bin, bin, key0, key1);
  }
  if (members > kFsCap) {
    // one key, too many ids: count along the ids
    const float x0 = fs_value(key0);
    const u64 w = r.weight(x0), nth = ids ? rest : (rest + w - 1) / w;
    if (out) {
      u64 mine = 0;
      for (int i = t; i < n; i += kFsThreads) mine += S.x[i] == x0;
      mine = fs_sum(S, mine);
      const u64* of = share(S, mine, rank, ctas);
      u64 skip = nth - 1;  // ids with this key before the one wanted
      for (uint32_t i = 0; i < rank; ++i) skip -= of[i];
      if (skip < mine) {  // (not where it fell below 0)
        // this CTA's: a thread a run of ids
        const int per = (n + kFsThreads - 1) / kFsThreads, lo = min(n, t * per),
                  hi = min(n, lo + per);
        u64 here = 0;
        for (int i = lo; i < hi; ++i) here += S.x[i] == x0;
        u64 k = skip - fs_before(S, here);
        for (int i = lo; i < hi && k < here; ++i)
          if (S.x[i] == x0 && k-- == 0) *out = id0 + i;
      }
    }
    return below + nth * w;
  }
  if (rank == 0) {
    if (members > kFsFew && key0 < key1) {
      // a list this long in parts first, and only the part that counts sorted
      const int shift = max(0, 24 - __clz(key1 - key0));
      if (t < 256) S.digit.put(t, 0, 0);
      if (t == 0) S.mine = 0;
      __syncthreads();
      for (int i = t; i < members; i += kFsThreads) {
        const uint32_t k = uint32_t(S.list[i] >> 32);
        S.digit.add((k - key0) >> shift, r.weight(fs_value(k)), true);
      }
      __syncthreads();
      const uint32_t d = uint32_t(fs_part(S, ids, &rest, &below));
      for (int i = t; i < members; i += kFsThreads) {
        const u64 e = S.list[i];
        if ((uint32_t(e >> 32) - key0) >> shift == d) S.run[atomicAdd(&S.mine, 1u)] = e;
      }
      __syncthreads();
      members = int(S.mine);
      for (int i = t; i < members; i += kFsThreads) S.list[i] = S.run[i];
      __syncthreads();
    }
    fs_sort(S, r, members);
    const int at = min(
        ids ? int(rest) - 1 : fs_reach(S, members, rest, [&](int i) { return S.run[i]; }),
        members - 1);
    if (t < int(ctas)) st_cluster(&S.answer, t, below + S.run[at]);
    if (out && t == 0) *out = int(~uint32_t(S.list[at]));
  }
  cluster_sync();
  return S.answer;
}

// The running weight that a share of `left` asks for: at least 1, at most all.
TTS_DEV u64 fs_target(double share, u64 left) {
  const double v = ceil(share * double(left));
  return v >= double(left) ? left : v > 1. ? u64(v) : 1ull;
}

struct FsArgs {
  FilterSampleRequest r;
  int per;  // ids a CTA holds
};

template <typename T>
__global__ void __launch_bounds__(kFsThreads, 2) filter_sample_kernel(const FsArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  FsSmem& S = *reinterpret_cast<FsSmem*>(smem_raw);
  const uint32_t rank = cluster_rank(), ctas = cluster_size();
  const int t = threadIdx.x, row = blockIdx.x / ctas;
  const int id0 = min(a.r.n, int(rank) * a.per), n = min(a.r.n - id0, a.per);
  const T* x = static_cast<const T*>(a.r.logits) + (size_t)row * a.r.ldl + id0;
  int* out = a.r.out + row;
  for (int b = t; b < kFsBins; b += kFsThreads) S.bin.put(b, 0, 0);
  if (t < 256) S.exp_table[t] = exp2(t / 256.);
  // ---- the row's part, once, and its maximum with the first id that has it
  u64 best = 0;
  float top = -INFINITY, bottom = INFINITY;
  int top_at = 0;
  const auto take = [&](int i, float f) {
    f = fs_clean(f);
    S.x[i] = f;
    if (f > top) top = f, top_at = i;
    if (f > -INFINITY) bottom = fminf(bottom, f);
  };
  // 16-byte loads from the first aligned element on
  constexpr int kVec = 16 / int(sizeof(T));
  const int head =
      min(n, int((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
  const int body = (n - head) / kVec;
  if (t < head) take(t, float(x[t]));
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  for (int i0 = t; i0 < body; i0 += kFsThreads * kFsLoads) {
    uint4 v[kFsLoads];
#pragma unroll
    for (int u = 0; u < kFsLoads; ++u)
      if (i0 + u * kFsThreads < body) v[u] = __ldcs(xv + i0 + u * kFsThreads);
#pragma unroll
    for (int u = 0; u < kFsLoads; ++u)
      if (i0 + u * kFsThreads < body) {
        const T* e = reinterpret_cast<const T*>(&v[u]);
#pragma unroll
        for (int w = 0; w < kVec; ++w)
          take(head + (i0 + u * kFsThreads) * kVec + w, float(e[w]));
      }
  }
  for (int i = head + body * kVec + t; i < n; i += kFsThreads) take(i, float(x[i]));
  if (t < 4 && n + t < (n + 3) / 4 * 4) S.x[n + t] = -INFINITY;
  if (top > -INFINITY) best = (u64(float_order_key(top)) << 32) | uint32_t(~(id0 + top_at));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 b = __shfl_xor_sync(0xffffffffu, best, o);
    best = b > best ? b : best;
  }
  if ((t & 31) == 0) S.part[t >> 5] = best;
  __syncthreads();
  for (int i = 0; i < kFsWarps; ++i) best = S.part[i] > best ? S.part[i] : best;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    bottom = fminf(bottom, __shfl_xor_sync(0xffffffffu, bottom, o));
  if ((t & 31) == 0) S.low[t >> 5] = bottom;
  __syncthreads();
  for (int i = 0; i < kFsWarps; ++i) bottom = fminf(bottom, S.low[i]);
  cluster_sync();  // every CTA of the row has started
  FsShare share;
  {
    if (t < int(ctas)) st_cluster(&S.floor[rank], t, __float_as_uint(bottom));
    const u64* of = share(S, best, rank, ctas);
    for (uint32_t i = 0; i < ctas; ++i) {
      best = of[i] > best ? of[i] : best;
      bottom = fminf(bottom, __uint_as_float(S.floor[i]));
    }
  }
  const float temp = a.r.temperature ? a.r.temperature[row] : 1.f;
  if (!best || !(temp > 0.f)) {  // no id can be picked, or the largest logit is
    if (rank == 0 && t == 0) *out = best ? int(~uint32_t(best)) : -1;
    return;
  }
  FsScale r;
  r.mx = fs_value(uint32_t(best >> 32));
  if (r.mx == INFINITY) {  // infinite logits share the draw
    for (int i = t; i < n; i += kFsThreads) S.x[i] = S.x[i] == INFINITY ? 0.f : -INFINITY;
    r.mx = bottom = 0.f;
    __syncthreads();
  }
  r.c = 1.4426950408889634 / double(temp);
  // the bins span what the row has, 45 octaves at most (weights behind them are 0)
  const double octaves = (double(r.mx) - double(bottom)) * r.c;
  r.per_bin = float(r.c * ((kFsBins - 1) / fmin(fmax(octaves, 1e-3), double(kFsOctaves))));
  r.table = S.exp_table;
  // ---- counts and weights by bin, of the whole row in each of its CTAs
  const int want = a.r.top_k ? a.r.top_k[row] : 0;
  const bool counts = want > 0 && want < a.r.n;  // only top-k needs them
  for (int i = t * 4; i < n; i += kFsThreads * 4) {
    const float4 v = *reinterpret_cast<const float4*>(S.x + i);  // padded to fours with -inf
    const float e[4] = {v.x, v.y, v.z, v.w};
    u64 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = r.weight(e[u]);  // side by side: a long chain each
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (e[u] > -INFINITY) S.bin.add(r.bin(e[u]), w[u], counts);
  }
  fs_join(S.bin, rank, ctas);
  {
    constexpr int kPer = kFsBins / kFsThreads;
    u64 w[kPer], c[kPer], ws = 0, cs = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int b = t * kPer + u;
      ws += w[u] = S.bin.weight(b);
      cs += c[u] = S.bin.count[b];
    }
    ws = fs_before(S, ws);
    cs = fs_before(S, cs);
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      ws += w[u], cs += c[u];
      S.bin.put(t * kPer + u, ws, uint32_t(cs));
    }
    __syncthreads();
  }
  // ---- the cuts, then the draw (the same in all CTAs up to here and after each step)
  u64 left = S.bin.weight(kFsBins - 1);
  const u64 all = left;
  bool top_k = counts && uint32_t(want) < S.bin.count[kFsBins - 1];
  const float p = a.r.top_p ? a.r.top_p[row] : 1.f;
  const bool top_p = p < 1.f;
  const float mp = a.r.min_p ? a.r.min_p[row] : 0.f;
  // weights from here on pass min-p (0: all)
  const u64 least = mp > 0.f ? u64(ceil(fmin(double(mp), 1.) * kFsOne)) : 0;
  const float draw = a.r.draws[row];
  const double u = draw > 0.f ? double(draw) : 0.;
  int m = kFsCap + 1;
  if (top_k) {
    const int last = fs_reach(S, kFsBins, u64(want), [&](int i) { return u64(S.bin.count[i]); });
    // ids of no weight change nothing
    top_k = (last ? S.bin.weight(last - 1) : 0) < all;
    if (top_k && S.bin.count[last] <= uint32_t(kFsCap))
      m = fs_gather(S, r, n, id0, rank, ctas, share, 0, last, 1, 0xffffffffu);
  }
  const auto run = [&](int i) { return S.run[i]; };
  if (m <= kFsCap) {
    // few ids left: the first CTA has them all
    if (rank > 0) return;
    fs_sort(S, r, m);
    m = want;
    left = S.run[m - 1];
    if (top_p) {
      m = fs_reach(S, m, fs_target(double(p), left), run) + 1;
      left = S.run[m - 1];
    }
    if (least) {
      u64 pass = 0;
      for (int i = t; i < m; i += kFsThreads)
        pass += S.run[i] - (i ? S.run[i - 1] : 0) >= least;
      m = max(1, int(fs_sum(S, pass)));
      left = S.run[m - 1];
    }
    const int at = fs_reach(S, m, fs_target(u, left), run);
    if (t == 0) *out = int(~uint32_t(S.list[min(at, m - 1)]));
    return;
  }
  if (top_k) left = fs_resolve(S, r, n, id0, rank, ctas, share, true, u64(want), nullptr);
  if (top_p)
    left = fs_resolve(S, r, n, id0, rank, ctas, share, false, fs_target(double(p), left), nullptr);
  if (least) {
    // whole bins pass up to the one before the threshold's neighbour; the three around it by id
    const int bin = min(kFsBins - 1, int(-log2f(fminf(mp, 1.f)) * float(double(r.per_bin) / r.c)));
    u64 pass = 0;
    fs_each(S, n, [&](int, float x) {
      if (abs(r.bin(x) - bin) > 1) return;
      const u64 w = r.weight(x);
      pass += w >= least ? w : 0;
    });
    const u64* of = share(S, fs_sum(S, pass), rank, ctas);
    pass = bin > 1 ? S.bin.weight(bin - 2) : 0;
    for (uint32_t i = 0; i < ctas; ++i) pass += of[i];
    left = pass < left ? pass : left;
  }
  fs_resolve(S, r, n, id0, rank, ctas, share, false, fs_target(u, left), out);
  cluster_sync();  // no CTA leaves while another may still write to it
}

template <typename T>
cudaError_t launch_as(const FilterSampleRequest& r, int device, cudaStream_t st) {
  // The fewest CTAs a row whose part of it leaves room for two of them on an SM, then twice as
  // many while the rows do not fill the SMs and a part stays at 2048 ids or more (8 rows of 32000:
  // 22.1 us, without that 28.4, down to 4096 only 23.7; 8 rows of 2048 in parts of 1024: 11.7 for
  // 10.2).
  const int sms = num_sms(device);
  int ctas = 1;
  while (ctas < kFsMaxCluster &&
         ((r.n + ctas - 1) / ctas > kFsTwo ||
          (long(r.rows) * ctas * 2 <= 2 * sms && (r.n + ctas - 1) / ctas >= 4096)))
    ctas *= 2;
  FsArgs a{r, ((r.n + ctas - 1) / ctas + 7) / 8 * 8};
  static_assert(2 * (sizeof(FsSmem) + 4 * kFsTwo + 1024) <= 228 * 1024, "two CTAs an SM");
  const size_t smem = sizeof(FsSmem) + sizeof(float) * a.per;
  {
    // the opt-in shared-memory limit is a per-device function attribute
    static std::mutex mu;
    static bool done[64] = {false};
    std::lock_guard<std::mutex> lock(mu);
    if (device >= 0 && device < 64 && !done[device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(filter_sample_kernel<T>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               int(sizeof(FsSmem) + sizeof(float) * (kFilterMaxN / kFsMaxCluster)));
      if (e != cudaSuccess) return e;
      done[device] = true;
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(r.rows) * ctas, 1, 1);
  cfg.blockDim = dim3(kFsThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, filter_sample_kernel<T>, a);
}

}  // namespace

cudaError_t launch_filter_sample(const FilterSampleRequest& r, int device, cudaStream_t st) {
  return r.f16 ? launch_as<__half>(r, device, st) : launch_as<float>(r, device, st);
}

}  // namespace tts
