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
// A bin with too many ids (equal logits) is narrowed by the bits of its keys.
//
// A weight is evaluated in 64 bits and held as an integer multiple of 2^-44: sums of up to 2^18
// of them are exact in 64 bits, so neither the order of the atomics nor the number of CTAs can
// change a pick.
#include <mutex>

#include "tts_common.cuh"
#include "tts_internal.h"

namespace tts {

namespace {

typedef unsigned long long u64;
constexpr int kFsThreads = 512;
constexpr int kFsWarps = kFsThreads / 32;
constexpr int kFsBins = 1024;
constexpr int kFsCap = 1024;     // ids the first CTA sorts at once
constexpr int kFsMaxCluster = 8;
constexpr float kFsOctaves = 45.f;  // below 2^-45 a weight is 0
constexpr double kFsPerOctave = (kFsBins - 1) / double(kFsOctaves);
constexpr int kFsTwo = 19456;    // ids in a CTA's part up to which two CTAs share an SM
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
  __device__ __forceinline__ void add(int i, u64 w) {
    atomicAdd(&count[i], 1u);
    if (!w) return;
    const uint32_t low = uint32_t(w), old = atomicAdd(&lo[i], low);
    const uint32_t up = uint32_t(w >> 32) + (old + low < old ? 1u : 0u);
    if (up) atomicAdd(&hi[i], up);
  }
};

struct FsSmem {
  FsSums<kFsBins> bin;          // by bin, then running
  FsSums<256> digit;            // by 8 bits of the keys, in a bin too full to sort
  u64 list[kFsCap];             // first CTA: gathered ids, key << 32 | ~id
  u64 run[kFsCap];              // their running weights
  double exp_table[256];        // 2^(i / 256)
  u64 part[kFsWarps];
  u64 best[kFsMaxCluster];      // by CTA: its maximum, key << 32 | ~id; later its share of a sum
  u64 answer;                   // what one thread, or the first CTA, found
  uint32_t filled;              // first CTA: ids gathered
  uint32_t keys[1];             // this CTA's part of the row
};

TTS_DEV uint32_t fs_key(float f) {  // 0: the id cannot be picked
  f += 0.f;                         // -0 counts as 0
  return f > -INFINITY ? float_order_key(f) : 0u;
}
TTS_DEV float fs_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// ---- shared memory of the cluster's CTAs
TTS_DEV uint32_t ld_cluster(const uint32_t* p, uint32_t cta) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr(p, cta)) : "memory");
  return v;
}
TTS_DEV u64 ld_cluster(const u64* p, uint32_t cta) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr(p, cta)) : "memory");
  return v;
}
TTS_DEV void st_cluster(uint32_t* p, uint32_t cta, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(p, cta)), "r"(v) : "memory");
}
TTS_DEV void st_cluster(u64* p, uint32_t cta, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_addr(p, cta)), "l"(v) : "memory");
}
TTS_DEV uint32_t add_cluster(uint32_t* p, uint32_t cta, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;"
               : "=r"(old)
               : "r"(cluster_addr(p, cta)), "r"(v)
               : "memory");
  return old;
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
  uint32_t top;       // the maximum's key
  TTS_DEV int bin(uint32_t key) const {  // grows as the key falls
    if (key == top) return 0;            // also where the maximum is infinite
    return min(kFsBins - 1, int((mx - fs_value(key)) * per_bin));
  }
  TTS_DEV u64 weight(uint32_t key) const {
    if (key == top) return u64(1) << 44;
    const double t = (double(fs_value(key)) - double(mx)) * c;
    if (!(t > -double(kFsOctaves))) return 0;
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
    return u64(__double_as_longlong(f + 4503599627370496.)) & 0xfffffffffffffull;
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
  for (int i = 0; i < int(threadIdx.x >> 5); ++i) r += S.part[i];
  return r;
}

// The first place at which a running sum (inclusive, `n` entries) reaches `target`: `n` if none.
template <typename F>
TTS_DEV int fs_reach(FsSmem& S, int n, u64 target, F sum_at) {
  u64 below = 0;
  for (int i = threadIdx.x; i < n; i += kFsThreads) below += sum_at(i) < target;
  return int(fs_sum(S, below));
}

// The sums of the row's CTAs, in all of them: each adds up a share of the entries.
template <int N>
TTS_DEV void fs_join(FsSums<N>& s, uint32_t rank, uint32_t ctas) {
  cluster_sync();
  if (ctas == 1) return;
  const int share = (N + int(ctas) - 1) / int(ctas), b0 = int(rank) * share;
  for (int b = b0 + int(threadIdx.x); b < min(N, b0 + share); b += kFsThreads) {
    u64 w = 0;
    uint32_t c = 0;
    for (uint32_t i = 0; i < ctas; ++i) {
      w += (u64(ld_cluster(&s.hi[b], i)) << 32) + ld_cluster(&s.lo[b], i);
      c += ld_cluster(&s.count[b], i);
    }
    for (uint32_t i = 0; i < ctas; ++i) {  // only this CTA reads or writes these entries
      st_cluster(&s.lo[b], i, uint32_t(w));
      st_cluster(&s.hi[b], i, uint32_t(w >> 32));
      st_cluster(&s.count[b], i, c);
    }
  }
  cluster_sync();
}

// The sum of v over the row's CTAs (v alike in a CTA's threads).
TTS_DEV u64 fs_sum_row(FsSmem& S, u64 v, uint32_t rank, uint32_t ctas) {
  if (ctas == 1) return v;
  cluster_sync();  // the last use of `best`
  if (threadIdx.x < ctas) st_cluster(&S.best[rank], threadIdx.x, v);
  cluster_sync();
  u64 r = 0;
  for (uint32_t i = 0; i < ctas; ++i) r += S.best[i];
  return r;
}

// Puts this CTA's ids of the given bins and keys into the first CTA's list.
TTS_DEV void fs_gather(FsSmem& S, const FsScale& r, int n, int id0, int bin0, int bin1,
                       uint32_t key0, uint32_t key1) {
  for (int i = threadIdx.x; i < n; i += kFsThreads) {
    const uint32_t k = S.keys[i];
    if (k < key0 || k > key1 || k == 0) continue;
    const int b = r.bin(k);
    if (b < bin0 || b > bin1) continue;
    const uint32_t at = add_cluster(&S.filled, 0, 1u);
    if (at < uint32_t(kFsCap)) st_cluster(&S.list[at], 0, (u64(k) << 32) | uint32_t(~(id0 + i)));
  }
  cluster_sync();
}
// First CTA: sorts the list by key, then id, and runs its weights up. Returns its length.
TTS_DEV int fs_sort(FsSmem& S, const FsScale& r) {
  const int t = threadIdx.x, m = min(int(S.filled), kFsCap);
  int size = 32;
  while (size < m) size *= 2;
  __syncthreads();
  if (t == 0) S.filled = 0;
  for (int i = m + t; i < size; i += kFsThreads) S.list[i] = 0;
  for (int k = 2; k <= size; k *= 2)  // bitonic, larger first
    for (int j = k / 2; j > 0; j /= 2) {
      __syncthreads();
      for (int e = t; e < size / 2; e += kFsThreads) {
        const int i = (e / j) * 2 * j + e % j;
        const u64 a = S.list[i], b = S.list[i + j];
        if ((a < b) == ((i & k) == 0)) S.list[i] = b, S.list[i + j] = a;
      }
    }
  __syncthreads();
  constexpr int kPer = kFsCap / kFsThreads;
  u64 w[kPer], sum = 0;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int i = t * kPer + u;
    w[u] = i < m ? r.weight(uint32_t(S.list[i] >> 32)) : 0;
    sum += w[u];
  }
  sum = fs_before(S, sum);
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    sum += w[u];
    S.run[t * kPer + u] = sum;
  }
  __syncthreads();
  return m;
}

// Where the running count (`ids`) or weight of the order reaches `target` (at least 1, at most
// all): the weight up to there, the id there included. With `out` that id goes there. All of the
// row's CTAs call it.
TTS_DEV u64 fs_resolve(FsSmem& S, const FsScale& r, int n, int id0, uint32_t rank, uint32_t ctas,
                       bool ids, u64 target, int* out) {
  const int t = threadIdx.x;
  const int bin = fs_reach(S, kFsBins, target, [&](int i) {
    return ids ? u64(S.bin.count[i]) : S.bin.weight(i);
  });
  u64 below = bin ? S.bin.weight(bin - 1) : 0;  // the weight of the ids before those looked at
  const uint32_t before = bin ? S.bin.count[bin - 1] : 0;
  uint32_t members = S.bin.count[bin] - before;
  u64 rest = target - (ids ? u64(before) : below);
  uint32_t key0 = 1, key1 = 0xffffffffu;
  for (int shift = 24; members > uint32_t(kFsCap) && shift >= 0; shift -= 8) {
    __syncthreads();
    if (t < 256) S.digit.put(t, 0, 0);
    __syncthreads();
    for (int i = t; i < n; i += kFsThreads) {
      const uint32_t k = S.keys[i];
      if (k < key0 || k > key1 || k == 0 || r.bin(k) != bin) continue;
      S.digit.add((k >> shift) & 255, r.weight(k));
    }
    fs_join(S.digit, rank, ctas);
    // every thread for itself: from the largest digit down
    int d = 255;
    for (; d > 0; --d) {
      const u64 w = S.digit.weight(d), step = ids ? u64(S.digit.count[d]) : w;
      if (step >= rest) break;
      rest -= step;
      below += w;
    }
    members = S.digit.count[d];
    const uint32_t prefix = shift == 24 ? 0u : key0 & ~((256u << shift) - 1u);
    key0 = prefix | (uint32_t(d) << shift);
    key1 = key0 | ((1u << shift) - 1u);
    cluster_sync();  // all CTAs have read the sums
  }
  if (members > uint32_t(kFsCap)) {
    // one key, too many ids: count along the ids
    const u64 w = r.weight(key0), nth = ids ? rest : (rest + w - 1) / w;
    if (out) {
      u64 mine = 0;
      for (int i = t; i < n; i += kFsThreads) mine += S.keys[i] == key0;
      mine = fs_sum(S, mine);
      fs_sum_row(S, mine, rank, ctas);
      u64 skip = nth - 1;  // ids with this key before the one wanted
      if (ctas > 1)
        for (uint32_t i = 0; i < rank; ++i) skip -= S.best[i];
      if (skip < mine) {  // (not where it fell below 0)
        // this CTA's: a thread a run of ids
        const int per = (n + kFsThreads - 1) / kFsThreads, lo = min(n, t * per),
                  hi = min(n, lo + per);
        u64 here = 0;
        for (int i = lo; i < hi; ++i) here += S.keys[i] == key0;
        u64 k = skip - fs_before(S, here);
        for (int i = lo; i < hi && k < here; ++i)
          if (S.keys[i] == key0 && k-- == 0) *out = id0 + i;
      }
    }
    return below + nth * w;
  }
  fs_gather(S, r, n, id0, bin, bin, key0, key1);
  if (rank == 0) {
    const int m = fs_sort(S, r);
    const int at =
        min(ids ? int(rest) - 1 : fs_reach(S, m, rest, [&](int i) { return S.run[i]; }), m - 1);
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
  if (t == 0) S.filled = 0;
  // ---- the row's part, once, and its maximum with the first id that has it
  u64 best = 0;
#pragma unroll 8
  for (int i = t; i < n; i += kFsThreads) {
    const uint32_t k = fs_key(float(x[i]));
    S.keys[i] = k;
    const u64 b = (u64(k) << 32) | uint32_t(~(id0 + i));
    best = k && b > best ? b : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 b = __shfl_xor_sync(0xffffffffu, best, o);
    best = b > best ? b : best;
  }
  if ((t & 31) == 0) S.part[t >> 5] = best;
  __syncthreads();
  for (int i = 0; i < kFsWarps; ++i) best = S.part[i] > best ? S.part[i] : best;
  cluster_sync();  // every CTA of the row has started
  if (t < int(ctas)) st_cluster(&S.best[rank], t, best);
  cluster_sync();
  for (uint32_t i = 0; i < ctas; ++i) best = S.best[i] > best ? S.best[i] : best;
  const float temp = a.r.temperature ? a.r.temperature[row] : 1.f;
  if (!best || !(temp > 0.f)) {  // no id can be picked, or the largest logit is
    if (rank == 0 && t == 0) *out = best ? int(~uint32_t(best)) : -1;
    return;
  }
  FsScale r;
  r.top = uint32_t(best >> 32);
  r.mx = fs_value(r.top);
  r.c = 1.4426950408889634 / double(temp);
  r.per_bin = float(r.c * kFsPerOctave);
  r.table = S.exp_table;
  // ---- counts and weights by bin, of the whole row in each of its CTAs
  for (int i = t; i < n; i += kFsThreads) {
    const uint32_t k = S.keys[i];
    if (!k) continue;
    S.bin.add(r.bin(k), r.weight(k));
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
  const uint32_t have = S.bin.count[kFsBins - 1];
  const int want = a.r.top_k ? a.r.top_k[row] : 0;
  bool top_k = want > 0 && uint32_t(want) < have;
  const float p = a.r.top_p ? a.r.top_p[row] : 1.f;
  const bool top_p = p < 1.f;
  const float mp = a.r.min_p ? a.r.min_p[row] : 0.f;
  // weights from here on pass min-p (0: all)
  const u64 least = mp > 0.f ? u64(ceil(fmin(double(mp), 1.) * kFsOne)) : 0;
  const float draw = a.r.draws[row];
  const double u = draw > 0.f ? double(draw) : 0.;
  int last = kFsBins;  // the bin that the first cut falls into
  if (top_k) {
    last = fs_reach(S, kFsBins, u64(want), [&](int i) { return u64(S.bin.count[i]); });
    // ids of no weight change nothing
    if ((last ? S.bin.weight(last - 1) : 0) == all) top_k = false, last = kFsBins;
  }
  if (!top_k && top_p)
    last = fs_reach(S, kFsBins, fs_target(double(p), left), [&](int i) { return S.bin.weight(i); });
  const auto run = [&](int i) { return S.run[i]; };
  if (last < kFsBins && S.bin.count[last] <= uint32_t(kFsCap)) {
    // few ids left: the first CTA takes them all
    fs_gather(S, r, n, id0, 0, last, 1, 0xffffffffu);
    if (rank > 0) return;
    int m = fs_sort(S, r);
    if (top_k) m = want;
    left = top_k ? S.run[m - 1] : all;
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
  if (top_k) left = fs_resolve(S, r, n, id0, rank, ctas, true, u64(want), nullptr);
  if (top_p)
    left = fs_resolve(S, r, n, id0, rank, ctas, false, fs_target(double(p), left), nullptr);
  if (least) {
    // whole bins pass up to the one before the threshold's neighbour; the three around it by id
    const int bin = min(kFsBins - 1, int(-log2f(fminf(mp, 1.f)) * float(kFsPerOctave)));
    u64 pass = 0;
    for (int i = t; i < n; i += kFsThreads) {
      const uint32_t k = S.keys[i];
      if (!k || abs(r.bin(k) - bin) > 1) continue;
      const u64 w = r.weight(k);
      pass += w >= least ? w : 0;
    }
    pass = fs_sum_row(S, fs_sum(S, pass), rank, ctas) + (bin > 1 ? S.bin.weight(bin - 2) : 0);
    left = pass < left ? pass : left;
  }
  fs_resolve(S, r, n, id0, rank, ctas, false, fs_target(u, left), out);
  cluster_sync();  // no CTA leaves while another may still write to it
}

template <typename T>
cudaError_t launch_as(const FilterSampleRequest& r, int device, cudaStream_t st) {
  // The fewest CTAs a row whose part of it leaves room for two of them on an SM, then twice as
  // many while the rows do not fill the SMs and a part stays at 2048 ids or more.
  const int sms = num_sms(device);
  int ctas = 1;
  while (ctas < kFsMaxCluster &&
         ((r.n + ctas - 1) / ctas > kFsTwo ||
          (long(r.rows) * ctas * 2 <= 2 * sms && (r.n + ctas - 1) / ctas >= 4096)))
    ctas *= 2;
  FsArgs a{r, (r.n + ctas - 1) / ctas};
  static_assert(2 * (sizeof(FsSmem) + 4 * kFsTwo + 1024) <= 228 * 1024, "two CTAs an SM");
  const size_t smem = sizeof(FsSmem) + sizeof(uint32_t) * a.per;
  {
    // the opt-in shared-memory limit is a per-device function attribute
    static std::mutex mu;
    static bool done[64] = {false};
    std::lock_guard<std::mutex> lock(mu);
    if (device >= 0 && device < 64 && !done[device]) {
      const cudaError_t e =
          cudaFuncSetAttribute(filter_sample_kernel<T>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               int(sizeof(FsSmem) + sizeof(uint32_t) * (kFilterMaxN / kFsMaxCluster)));
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
